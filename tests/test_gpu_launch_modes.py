"""The one-call launch path under torch's modes: outputs that torch would show to a dispatch mode, or fill, still are."""
import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

from pyptx_b200.examples.blackwell.fp8_gemm import build_fp8_grouped_gemm_varlen, build_fp8_quantize
from pyptx_b200.examples.blackwell.grouped_gemm import build_grouped_gemm_varlen
from pyptx_b200.examples.blackwell.rms_norm import build_rms_norm

pytestmark = pytest.mark.gpu


class Seen(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.calls = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        out = func(*args, **(kwargs or {}))
        self.calls.append((func, out))
        return out


def test_a_dispatch_mode_sees_the_allocation():
    k = build_rms_norm(16, 512)
    x, w = torch.randn(16, 512, device="cuda"), torch.randn(512, device="cuda")
    want = k(x, w)
    for _ in range(2):
        with Seen() as mode:
            out = k(x, w)
        assert torch.equal(out, want)
        made = [o for f, o in mode.calls if f is torch.ops.aten.empty.memory_format]
        assert len(made) == 1 and made[0].data_ptr() == out.data_ptr()
    assert k._launcher.fast((x, w)) is not None                # and outside of it the one-call path is back


@pytest.fixture
def filled():
    before = torch.are_deterministic_algorithms_enabled(), torch.utils.deterministic.fill_uninitialized_memory
    torch.use_deterministic_algorithms(True)
    torch.utils.deterministic.fill_uninitialized_memory = True
    yield
    torch.use_deterministic_algorithms(before[0])
    torch.utils.deterministic.fill_uninitialized_memory = before[1]


def _grouped_inputs(kind):
    G, M, N, K = 2, 512, 256, 128
    if kind == "bf16":
        k = build_grouped_gemm_varlen(G, M, N, K)
        ins = [torch.ones(M, K, device="cuda").bfloat16(), torch.ones(G * N, K, device="cuda").bfloat16()]
    else:
        k = build_fp8_grouped_gemm_varlen(G, M, N, K)
        ins = [torch.ones(M, K, device="cuda").to(torch.float8_e4m3fn), torch.ones(M, 1, device="cuda"),
               torch.ones(G * N, K, device="cuda").to(torch.float8_e4m3fn), torch.ones(G * N // 128, 1, device="cuda")]
    return k, ins + [torch.tensor([0, 128, 256], dtype=torch.int32, device="cuda")]


@pytest.mark.parametrize("kind", ["bf16", "fp8"])
def test_rows_that_are_left_unwritten_are_filled(kind, filled):
    k, ins = _grouped_inputs(kind)
    for _ in range(3):
        out = k(*ins)
        assert (out[:256] == 128.0).all() and torch.isnan(out[256:]).all()
        del out
    torch.utils.deterministic.fill_uninitialized_memory = False
    assert k._launcher.fast(tuple(ins)) is not None


def test_eight_bit_outputs_under_the_fill(filled):
    x = torch.randn(64, 256, device="cuda").bfloat16()
    q = build_fp8_quantize(64, 256)
    a, b = q(x), q(x)
    torch.use_deterministic_algorithms(False)
    for want, first, second in zip(q(x), a, b):
        assert torch.equal(first.float(), want.float()) and torch.equal(second.float(), want.float())
