"""The one-call launch path of kernels with static shapes: same results and same refusals as the checking
path, call after call."""
import pytest
import torch

from pyptx_b200 import _native
from pyptx_b200.examples.blackwell import moe
from pyptx_b200.examples.blackwell.rms_norm import build_rms_norm
from pyptx_b200.examples.blackwell.backward import build_rms_norm_bwd

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def kernel():
    k = build_rms_norm(16, 512)
    k(torch.randn(16, 512, device="cuda"), torch.randn(512, device="cuda"))      # the first call makes the launcher
    assert k._launcher.fast is not None
    return k


def test_results_equal_the_checking_path(kernel):
    x, w = torch.randn(16, 512, device="cuda"), torch.randn(512, device="cuda")
    fast, kernel._launcher.fast = kernel._launcher.fast, None
    try:
        slow = kernel(x, w)
    finally:
        kernel._launcher.fast = fast
    assert torch.equal(kernel(x, w), slow)
    assert torch.equal(kernel(torch.nn.Parameter(x), w.requires_grad_()), slow)
    with torch.inference_mode():
        out = kernel(x, w)
        assert out.is_inference() and torch.equal(out, slow)


def test_scratch_and_several_outputs_come_back_as_a_tuple():
    k = build_rms_norm_bwd(64, 256)
    ins = [torch.randn(64, 256, device="cuda"), torch.randn(256, device="cuda"), torch.randn(64, 256, device="cuda")]
    first, second = k(*ins), k(*ins)
    assert isinstance(second, tuple) and len(second) == 2 and k.scratch_bytes > 0
    assert all(torch.equal(a, b) and a.shape == b.shape and a.dtype == b.dtype for a, b in zip(first, second))


@pytest.mark.parametrize("bad,error,message", [
    (lambda x, w: (x.cpu(), w), ValueError, "no CPU path"),
    (lambda x, w: (x, w.cpu()), ValueError, "input 1 is on cpu"),
    (lambda x, w: (x.half(), w), TypeError, "dtype"),
    (lambda x, w: (x.t().contiguous().t(), w), ValueError, "not contiguous"),
    (lambda x, w: (x[:8], w), ValueError, "expected 16, got 8"),
    (lambda x, w: (x, 3), TypeError, "int"),
    (lambda x, w: (x,), TypeError, "expected 2 input arrays"),
    (lambda x, w: (x, torch.cat([w, w])[1:513]), RuntimeError, "16-byte aligned"),
])
def test_refusals_stay_the_same_after_good_calls(kernel, bad, error, message):
    x, w = torch.randn(16, 512, device="cuda"), torch.randn(512, device="cuda")
    kernel(x, w)
    with pytest.raises(error, match=message):
        kernel(*bad(x, w))
    kernel(x, w)


def test_a_destroyed_handle_raises():
    k = build_rms_norm(8, 256)
    x, w = torch.randn(8, 256, device="cuda"), torch.randn(256, device="cuda")
    k(x, w)
    assert _native.load().pb200_destroy(k.handle) == 0
    with pytest.raises(RuntimeError, match="unknown handle"):
        k(x, w)


def test_more_inputs_than_specs_are_ignored_as_before(kernel):
    x, w = torch.randn(16, 512, device="cuda"), torch.randn(512, device="cuda")
    assert torch.equal(kernel(x, w, None), kernel(x, w))


def test_side_stream_and_threads():
    """The current stream counts, and concurrent host threads do not disturb one another."""
    import threading

    T, k, E = 512, 4, 16
    route = moe.build_moe_route(T, k, E, block=8)
    ids = [torch.randint(0, E, (T, k), dtype=torch.int32, device="cuda") for _ in range(4)]
    want = [route(i) for i in ids]
    got = [[] for _ in ids]

    def work(n):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(50):
                got[n].append(route(ids[n]))
        stream.synchronize()

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(n,)) for n in range(len(ids))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for n, outs in enumerate(got):
        assert len(outs) == 50
        for out in outs:
            assert all(torch.equal(a, b) for a, b in zip(out, want[n]))


def test_threads_that_route_different_sizes():
    """Shared memory differs between these (one needs 184 KB, one 54 KB, one 164 KB, one 38 KB in two launches); none may
    narrow another's limit."""
    import threading

    shapes = [(32768, 1, 1024), (2048, 1, 255), (16384, 1, 1000), (40000, 1, 300)]
    routes = [moe.build_moe_route(T, k, E, block=1) for T, k, E in shapes]
    ids = [torch.randint(0, E, (T, k), dtype=torch.int32, device="cuda") for T, k, E in shapes]
    torch.cuda.synchronize()
    errors, counts = [], [0] * len(shapes)
    start = threading.Barrier(len(shapes))

    def work(n):
        try:
            with torch.cuda.stream(torch.cuda.Stream()) as _:
                start.wait()
                for _ in range(300):
                    row_of, entry_of, offsets = routes[n](ids[n])
                torch.cuda.current_stream().synchronize()
            order = torch.sort(ids[n].flatten(), stable=True).indices
            assert torch.equal(entry_of.long(), order)
            counts[n] += 1
        except Exception as exc:  # noqa: BLE001
            errors.append(exc)

    threads = [threading.Thread(target=work, args=(n,)) for n in range(len(shapes))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    assert counts == [1] * len(shapes)


@pytest.mark.parametrize("kind", ["gemm", "fp8_gemm", "rms_norm"])
def test_a_thread_whose_first_cuda_call_is_a_launch(kind):
    """The raw entry from a host thread that has made no CUDA call (and so has no context bound)."""
    import threading

    from pyptx_b200.examples.blackwell.fp8_gemm import build_fp8_gemm
    from pyptx_b200.examples.blackwell.gemm_highperf_blackwell import build_gemm

    if kind == "gemm":
        k, ins = build_gemm(128, 256, 64), [torch.ones(128, 64, device="cuda").bfloat16(), torch.ones(256, 64, device="cuda").bfloat16()]
    elif kind == "fp8_gemm":
        one = torch.ones(64, 128, device="cuda")
        k, ins = build_fp8_gemm(64, 64, 128), [one.to(torch.float8_e4m3fn), one[:, :1].contiguous(), one.to(torch.float8_e4m3fn),
                                              torch.ones(1, 1, device="cuda")]
    else:
        k, ins = build_rms_norm(16, 512), [torch.ones(16, 512, device="cuda"), torch.ones(512, device="cuda")]
    want = k(*ins)
    out = torch.zeros_like(want)
    ptrs = [t.data_ptr() for t in ins] + [out.data_ptr()]
    torch.cuda.synchronize()
    errors = []

    def work():
        try:
            _native.launch_raw(k.handle, 0, ptrs)
        except Exception as exc:  # noqa: BLE001
            errors.append(exc)

    thread = threading.Thread(target=work)
    thread.start()
    thread.join()
    torch.cuda.synchronize()
    assert not errors, errors
    assert torch.equal(out, want)
