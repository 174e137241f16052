"""GPU parity of the mixture-of-experts token movement and the 8-bit quantisation against float64 loops
(oracle/formulas.py): integer maps and copies are equal, sums lie within their rounding bounds."""
import pytest
import torch

from oracle import formulas
from pyptx_b200.examples.blackwell import moe
from pyptx_b200.examples.blackwell.fp8_gemm import build_fp8_quantize
from pyptx_b200.types import bf16, f32, s64

pytestmark = pytest.mark.gpu

TORCH = {"bf16": torch.bfloat16, "f32": torch.float32}
PTX = {"bf16": bf16, "f32": f32}
U32 = 2.0 ** -24                                   # half a step of f32, relative
HALF_STEP = {"bf16": 2.0 ** -8, "f32": 2.0 ** -24}


def _ids(T, k, E, seed, dropped=0.0):
    g = torch.Generator().manual_seed(seed)
    ids = (torch.randn(E, generator=g) + torch.rand(T, E, generator=g)).topk(k, dim=-1).indices.to(torch.int32)
    away = torch.rand(T, k, generator=g) < dropped
    return torch.where(away, torch.full_like(ids, -1), ids)


def _check_route(ids, E, block, rows=None, ids_dtype=None):
    T, k = ids.shape
    kw = {} if ids_dtype is None else {"ids_dtype": ids_dtype}
    kernel = moe.build_moe_route(T, k, E, block=block, rows=rows, **kw)
    R = kernel.meta["rows"]
    got = kernel(ids.cuda())
    want = formulas.moe_route_ref(ids, E, block, R)
    for name, a, b in zip(("row_of", "entry_of", "offsets"), got, want):
        assert a.dtype == torch.int32 and torch.equal(a.cpu(), b), name
    return got


# ---- route -----------------------------------------------------------------------------------

@pytest.mark.parametrize("T,k,E,block", [
    (1, 1, 1, 1), (1, 8, 256, 128), (7, 2, 3, 1), (33, 4, 16, 8), (256, 8, 64, 128), (1000, 3, 10, 16),
    (2049, 1, 1024, 128), (4096, 8, 128, 1), (8192, 4, 1024, 8), (16000, 2, 61, 128),      # 1 to 8 CTAs
    (32769, 1, 1, 1), (5000, 32, 32, 100), (8192, 8, 256, 128), (40000, 8, 60, 128), (9000, 32, 1024, 1),      # two launches
    (512, 1, 128, 1), (64, 8, 127, 128), (513, 1, 128, 4), (64, 8, 129, 1), (16, 32, 33, 1024),
    (256, 1, 128, 1), (257, 1, 128, 1), (32, 8, 128, 128), (32, 8, 129, 128),              # few warps, and just not
])
@pytest.mark.parametrize("dropped", [0.0, 0.4])
def test_route_matches_stable_sort(T, k, E, block, dropped):
    _check_route(_ids(T, k, E, T + k + E, dropped), E, block)


@pytest.mark.parametrize("T,k", [(1, 1), (50, 4), (6000, 4)])
def test_route_with_nothing_to_place(T, k):
    ids = torch.full((T, k), -1, dtype=torch.int32)
    row_of, entry_of, offsets = _check_route(ids, 8, 16)
    assert (row_of == -1).all() and (entry_of == -1).all() and (offsets == 0).all()


def test_route_one_expert_takes_all_and_repeats():
    _check_route(torch.full((700, 4), 5, dtype=torch.int32), 8, 128)              # the same expert twice in a token
    _check_route(torch.full((9000, 8), 0, dtype=torch.int32), 1, 1)
    _check_route(torch.full((9000, 8), 1023, dtype=torch.int32), 1024, 128)


def test_route_drops_ids_out_of_range():
    ids = torch.tensor([[0, 3, 4], [-5, 2 ** 31 - 1, -2 ** 31], [1, 1, 2]], dtype=torch.int32)
    row_of, _, offsets = _check_route(ids, 4, 1)
    assert (row_of.cpu()[1] == -1).all() and offsets.tolist() == [0, 1, 3, 4, 5]
    wide = torch.tensor([[0, 2 ** 32, 1], [2 ** 32 + 1, -1, 3], [2 ** 62, -2 ** 62, 2]], dtype=torch.int64)
    row_of, _, _ = _check_route(wide, 4, 8, ids_dtype=s64)
    assert row_of.cpu()[0, 1] == -1 and row_of.cpu()[1, 0] == -1


@pytest.mark.parametrize("T,k,E,block,rows", [(64, 4, 8, 16, 16), (64, 4, 8, 16, 160), (3000, 8, 64, 128, 12800),
                                              (40000, 8, 60, 1, 100000), (5, 1, 4, 1, 4000)])
def test_route_with_its_own_row_count(T, k, E, block, rows):
    """Fewer rows than entries: the rest is dropped and offsets are clipped.  More: the tail is unowned."""
    row_of, entry_of, offsets = _check_route(_ids(T, k, E, rows), E, block, rows)
    assert int(offsets.max()) <= rows and entry_of.numel() == rows


# ---- dispatch --------------------------------------------------------------------------------

MOVES = [(1, 1, 1, 8, 1), (1, 8, 16, 64, 128), (5, 3, 4, 1000, 8), (77, 4, 9, 4104, 16), (300, 2, 64, 16384, 1),
         (1500, 6, 40, 264, 128), (20, 32, 33, 512, 4)]


@pytest.mark.parametrize("T,k,E,H,block", MOVES)
@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("dropped", [0.0, 0.5])
def test_dispatch_and_its_gradient(T, k, E, H, block, kind, dropped):
    R = moe.moe_rows(T, k, E, block)
    row_of, entry_of, _ = moe.build_moe_route(T, k, E, block=block)(_ids(T, k, E, H, dropped).cuda())
    g = torch.Generator().manual_seed(T * 31 + H)
    x = torch.randn(T, H, generator=g).to(TORCH[kind])
    rows = moe.build_moe_dispatch(T, k, R, H, dtype=PTX[kind])(x.cuda(), row_of, entry_of)
    assert torch.equal(rows.cpu(), formulas.moe_dispatch_ref(x, entry_of.cpu(), k))
    d_rows = torch.randn(R, H, generator=g).to(TORCH[kind])
    d_rows[entry_of.cpu() < 0] = float("nan")                  # rows nobody owns are not read
    dx = moe.build_moe_dispatch_bwd(T, k, R, H, dtype=PTX[kind])(row_of, d_rows.cuda()).cpu().double()
    want, mag = formulas.moe_combine_ref(d_rows, None, row_of.cpu())
    assert ((dx - want).abs() <= HALF_STEP[kind] * want.abs() + 2 * k * U32 * mag).all()


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("T,k,E,H,block", [(1, 1, 1, 16, 1), (3, 2, 8, 128, 1), (16, 8, 128, 4096, 1), (200, 4, 9, 1040, 32),
                                           (2500, 2, 5, 2064, 128)])
def test_dispatch_fp8_equals_quantised_dispatch(T, k, E, H, block, kind):
    R = moe.moe_rows(T, k, E, block)
    row_of, entry_of, _ = moe.build_moe_route(T, k, E, block=block)(_ids(T, k, E, H, 0.2).cuda())
    x = (torch.randn(T, H, generator=torch.Generator().manual_seed(H)) * 3).to(TORCH[kind])
    q, scale = moe.build_moe_dispatch_fp8(T, k, R, H, in_dtype=PTX[kind])(x.cuda(), row_of, entry_of)
    wq, ws = formulas.fp8_quantize_ref(x, 1)
    assert torch.equal(q.cpu().double(), formulas.moe_dispatch_ref(wq, entry_of.cpu(), k))
    assert torch.equal(scale.cpu().double(), formulas.moe_dispatch_ref(ws, entry_of.cpu(), k))


# ---- combine ---------------------------------------------------------------------------------

@pytest.mark.parametrize("T,k,E,H,block", MOVES)
@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("dropped", [0.0, 0.5, 1.0])
def test_combine_and_its_gradient(T, k, E, H, block, kind, dropped):
    R = moe.moe_rows(T, k, E, block)
    row_of, entry_of, _ = moe.build_moe_route(T, k, E, block=block)(_ids(T, k, E, H, dropped).cuda())
    g = torch.Generator().manual_seed(T * 37 + H)
    y = torch.randn(R, H, generator=g).to(TORCH[kind])
    y[entry_of.cpu() < 0] = float("inf")                       # rows nobody owns are not read
    w = torch.rand(T, k, generator=g) - 0.3
    w[row_of.cpu() < 0] = float("nan")                         # nor are dropped entries' weights
    out = moe.build_moe_combine(T, k, R, H, dtype=PTX[kind])(y.cuda(), w.cuda(), row_of).cpu().double()
    want, mag = formulas.moe_combine_ref(y, w, row_of.cpu())
    assert ((out - want).abs() <= HALF_STEP[kind] * want.abs() + 2 * k * U32 * mag).all()

    dout = torch.randn(T, H, generator=g).to(TORCH[kind])
    d_rows, d_w = moe.build_moe_combine_bwd(T, k, R, H, dtype=PTX[kind])(y.cuda(), w.cuda(), row_of, entry_of, dout.cuda())
    want_rows, want_w, mag_w = formulas.moe_combine_bwd_ref(y, w, row_of.cpu(), dout)
    # one f32 product (a rounding of its own when the rows are bf16), rounded to the rows' type
    assert ((d_rows.cpu().double() - want_rows).abs() <= (HALF_STEP[kind] + 2 * U32) * want_rows.abs()).all()
    assert ((d_w.cpu().double() - want_w).abs() <= H * U32 * mag_w).all()
    assert (d_w.cpu()[row_of.cpu() < 0] == 0).all()


def test_combine_passes_special_values_of_owned_rows():
    T, k, E, H = 4, 2, 4, 64
    row_of, entry_of, _ = moe.build_moe_route(T, k, E, block=1)(torch.tensor([[0, 1], [2, 3], [1, 0], [3, 2]], dtype=torch.int32).cuda())
    y = torch.ones(T * k, H)
    y[int(row_of[1, 0]), 3] = float("nan")
    y[int(row_of[2, 1]), 5] = float("-inf")
    out = moe.build_moe_combine(T, k, T * k, H, dtype=f32)(y.cuda(), torch.ones(T, k).cuda(), row_of).cpu()
    assert torch.isnan(out[1, 3]) and out[2, 5] == float("-inf") and torch.isfinite(out).sum() == T * H - 2


def test_maps_that_point_outside_are_ignored():
    """Maps from elsewhere: rows outside [0, R) count as dropped, nothing outside the buffers is touched."""
    T, k, R, H = 6, 2, 8, 64
    row_of = torch.tensor([[0, 8], [-7, 1], [2 ** 31 - 1, 2], [3, -2 ** 31], [4, 5], [6, 7]], dtype=torch.int32)
    entry_of = torch.full((R,), -1, dtype=torch.int32)
    legal = torch.where((row_of >= 0) & (row_of < R), row_of, torch.full_like(row_of, -1))
    for t in range(T):
        for j in range(k):
            if legal[t, j] >= 0:
                entry_of[legal[t, j]] = t * k + j
    x = torch.randn(T, H)
    rows = moe.build_moe_dispatch(T, k, R, H, dtype=f32)(x.cuda(), row_of.cuda(), entry_of.cuda())
    assert torch.equal(rows.cpu(), formulas.moe_dispatch_ref(x, entry_of, k))
    w = torch.rand(T, k)
    out = moe.build_moe_combine(T, k, R, H, dtype=f32)(rows, w.cuda(), row_of.cuda()).cpu().double()
    want, mag = formulas.moe_combine_ref(rows.cpu(), w, legal)
    assert ((out - want).abs() <= U32 * want.abs() + 2 * k * U32 * mag).all()
    q, _ = moe.build_moe_dispatch_fp8(T, k, R, H, in_dtype=f32)(x.cuda(), row_of.cuda(), entry_of.cuda())
    assert torch.equal(q.cpu().double(), formulas.moe_dispatch_ref(formulas.fp8_quantize_ref(x, 1)[0], entry_of, k))
    d_rows, d_w = moe.build_moe_combine_bwd(T, k, R, H, dtype=f32)(rows, w.cuda(), row_of.cuda(), entry_of.cuda(), x.cuda())
    want_rows, want_w, mag_w = formulas.moe_combine_bwd_ref(rows.cpu(), w, legal, x)
    assert ((d_rows.cpu().double() - want_rows).abs() <= 3 * U32 * want_rows.abs()).all()
    assert ((d_w.cpu().double() - want_w).abs() <= H * U32 * mag_w).all()


def test_rows_beyond_two_to_the_31_elements():
    """2.2e9 elements of sorted rows: the last ones are addressed with 64-bit offsets in every direction."""
    T, k, R, H = 6, 2, 540000, 4096
    row_of = torch.tensor([[0, 539999], [524287, 524288], [3, 4], [539998, 1], [300000, 2], [-1, 400000]], dtype=torch.int32)
    entry_of = torch.full((R,), -1, dtype=torch.int32)
    for i, r in enumerate(row_of.reshape(-1).tolist()):
        if r >= 0:
            entry_of[r] = i
    row_of, entry_of = row_of.cuda(), entry_of.cuda()
    x, w = torch.randn(T, H).to(torch.bfloat16).cuda(), torch.rand(T, k).cuda()
    rows = moe.build_moe_dispatch(T, k, R, H)(x, row_of, entry_of)
    for t in range(T):
        for j in range(k):
            if row_of[t, j] >= 0:
                assert torch.equal(rows[int(row_of[t, j])], x[t])
    assert (rows[539990:539998] == 0).all() and (rows[524289:524400] == 0).all()
    dx = moe.build_moe_dispatch_bwd(T, k, R, H)(row_of, rows)
    kept = (row_of >= 0).sum(dim=1, keepdim=True)
    assert torch.equal(dx, (x.float() * kept).to(torch.bfloat16))
    d_rows, d_w = moe.build_moe_combine_bwd(T, k, R, H)(rows, w, row_of, entry_of, x)
    assert torch.equal(d_rows[539999].float(), (w[0, 1] * x[0].float()).to(torch.bfloat16).float())
    assert (d_w[5, 0] == 0) and (d_w[5, 1] - x[5].double().square().sum()).abs() <= H * U32 * x[5].double().square().sum()
    q, scale = moe.build_moe_dispatch_fp8(T, k, R, H)(x, row_of, entry_of)
    wq, ws = formulas.fp8_quantize_ref(x.cpu(), 1)
    assert torch.equal(q[539999].cpu().double(), wq[0]) and torch.equal(scale[539998].cpu().double(), ws[3])
    assert (q[524289:524400].float() == 0).all() and (scale[524289:524400] == 0).all()


# ---- quantisation ----------------------------------------------------------------------------

@pytest.mark.parametrize("M,K", [(1, 16), (1, 4096), (3, 144), (127, 272), (129, 2064), (1000, 1040), (5000, 256)])
@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_is_exact(M, K, kind, block_rows):
    g = torch.Generator().manual_seed(M * 3 + K)
    x = (torch.randn(M, K, generator=g) * torch.exp(4 * torch.randn(M, 1, generator=g))).to(TORCH[kind])
    q, scale = build_fp8_quantize(M, K, block_rows=block_rows, in_dtype=PTX[kind])(x.cuda())
    wq, ws = formulas.fp8_quantize_ref(x, block_rows)
    assert q.dtype == torch.float8_e4m3fn and q.shape == (M, K)
    assert torch.equal(scale.cpu().double(), ws) and torch.equal(q.cpu().double(), wq)


@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_the_longest_row(block_rows):
    """2^31 - 65536 columns, the most that is accepted."""
    K = 2 ** 31 - 65536
    x = torch.zeros(1, K, dtype=torch.bfloat16, device="cuda")
    at = [5, 2 ** 30, K - 200, K - 1]
    for i, c in enumerate(at):
        x[0, c] = 448.0 * 2 ** i
    q, scale = build_fp8_quantize(1, K, block_rows=block_rows)(x)
    assert int(torch.count_nonzero(q.view(torch.uint8).view(torch.int32))) == len(at)
    assert int((scale > 2.0 ** -100).sum()) == len(at)
    for i, c in enumerate(at):
        assert float(q[0, c]) == 448.0 and float(scale[0, c // 128]) == 2.0 ** i


@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_special_blocks(block_rows):
    """All zeros, the smallest numbers, the largest, a NaN, an infinity: one 128-column block each."""
    M, K = 128, 128 * 6
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(1))
    x[:, :128] = 0.0
    x[:, 128:256] *= 1e-38
    x[:, 256:384] = x[:, 256:384].clamp(-1, 1) * 3.4e38
    x[5, 400] = float("nan")
    x[7, 600] = float("inf")
    q, scale = build_fp8_quantize(M, K, block_rows=block_rows, in_dtype=f32)(x.cuda())
    q, scale = q.cpu().double(), scale.cpu().double()
    wq, ws = formulas.fp8_quantize_ref(x, block_rows)
    assert torch.equal(scale, ws)
    for c in (0, 1, 2, 5):
        assert torch.equal(q[:, c * 128:(c + 1) * 128], wq[:, c * 128:(c + 1) * 128]), c
    nan = torch.zeros(M, 128, dtype=torch.bool)
    nan[5, 16] = True
    assert torch.equal(torch.isnan(q[:, 384:512]), nan)
    assert torch.equal(q[:, 384:512][~nan], wq[:, 384:512][~nan])
    back = q[:, 512:640] * scale[:, 4:5].repeat_interleave(block_rows, dim=0)[:M]
    assert torch.isnan(back[7]).all()
    if block_rows == 1:
        assert torch.isfinite(back[:7]).all()


# ---- autograd, graphs, streams ---------------------------------------------------------------

def test_autograd_against_differences():
    """The layer is linear in x, rows and weights, so a central difference with step 1 is the derivative
    up to rounding."""
    T, k, E, H, block = 40, 3, 6, 96, 4
    R = moe.moe_rows(T, k, E, block)
    row_of, entry_of, _ = moe.build_moe_route(T, k, E, block=block)(_ids(T, k, E, 3, 0.2).cuda())
    dispatch = moe.build_differentiable_moe_dispatch(T, k, R, H, dtype=f32)
    combine = moe.build_differentiable_moe_combine(T, k, R, H, dtype=f32)
    g = torch.Generator(device="cuda").manual_seed(9)
    x = torch.randn(T, H, generator=g, device="cuda", requires_grad=True)
    w = torch.rand(T, k, generator=g, device="cuda", requires_grad=True)
    factor = torch.randn(R, 1, generator=g, device="cuda")
    dout = torch.randn(T, H, generator=g, device="cuda")

    def layer(x_, w_):
        return combine(dispatch(x_, row_of, entry_of) * factor, w_, row_of, entry_of)

    gx, gw = torch.autograd.grad(layer(x, w), (x, w), dout)
    with torch.no_grad():
        for value, grad, other in ((x, gx, lambda v: layer(v, w)), (w, gw, lambda v: layer(x, v))):
            d = torch.randn(value.shape, generator=g, device="cuda")
            up, down = (other(value + d).double() * dout).sum(), (other(value - d).double() * dout).sum()
            slope = (grad.double() * d).sum()
            size = (grad.double() * d).abs().sum() + (other(value).double() * dout).abs().sum()
            assert abs((up - down) / 2 - slope) <= 64 * U32 * size


def test_expanded_gradients_and_shared_leaves():
    T, k, E, H = 12, 2, 3, 64
    R = T * k
    row_of, entry_of, _ = moe.build_moe_route(T, k, E, block=1)(_ids(T, k, E, 5).cuda())
    dispatch = moe.build_differentiable_moe_dispatch(T, k, R, H, dtype=f32)
    x = torch.randn(T, H, device="cuda", requires_grad=True)
    (dispatch(x, row_of, entry_of).sum() + 2 * dispatch(x, row_of, entry_of).sum()).backward()
    assert torch.equal(x.grad, torch.full_like(x, 3.0 * k))


def test_graph_replay_with_new_routing():
    """One captured graph serves every routing outcome; two replays of different ids, and another stream."""
    T, k, E, H, block = 300, 4, 12, 512, 16
    R = moe.moe_rows(T, k, E, block)
    route = moe.build_moe_route(T, k, E, block=block)
    dispatch = moe.build_moe_dispatch(T, k, R, H)
    combine = moe.build_moe_combine(T, k, R, H)
    ids = _ids(T, k, E, 1).cuda()
    x = torch.randn(T, H, device="cuda").to(torch.bfloat16)
    w = torch.full((T, k), 1.0 / k, device="cuda")

    def step():
        row_of, entry_of, _ = route(ids)
        rows = dispatch(x, row_of, entry_of)
        return row_of, rows, combine(rows, w, row_of)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in (2, 3):
        ids.copy_(_ids(T, k, E, seed, 0.3).cuda())
        graph.replay()
        eager = step()
        torch.cuda.synchronize()
        for a, b in zip(captured, eager):
            assert torch.equal(a, b)


def test_compiled_route_and_dispatch():
    T, k, E, H = 64, 2, 8, 128
    route = moe.build_moe_route(T, k, E, block=8)
    R = route.meta["rows"]
    dispatch = moe.build_moe_dispatch_fp8(T, k, R, H)
    ids, x = _ids(T, k, E, 4).cuda(), torch.randn(T, H, device="cuda").to(torch.bfloat16)

    def step(ids_, x_):
        row_of, entry_of, offsets = route(ids_)
        return (row_of, offsets, *dispatch(x_, row_of, entry_of))

    for a, b in zip(torch.compile(step)(ids, x), step(ids, x)):
        assert torch.equal(a.float(), b.float())
