"""Mixture-of-experts movement at the edges of what it accepts."""
import pytest
import torch

from oracle import formulas
from pyptx_b200 import _native
from pyptx_b200.examples.blackwell import moe

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [8, 32768, 150000])
def test_route_with_the_most_rows_that_are_accepted(T):
    """2^31 - 65536 rows: a row counter that takes one step of the grid past the last row leaves 32 bits (150000
    entries are placed by 147 CTAs of 1024 threads, a step of 150528 rows; one cluster's is 8192 at most).  A
    wrapped counter would start again at -2^31, so the 2^31 words before ``entry_of`` are looked at too."""
    E, rows, guard = 8, 2 ** 31 - 65536, 2 ** 31
    route = moe.build_moe_route(T, 1, E, block=1, rows=rows)
    ids = torch.randint(0, E, (T, 1), generator=torch.Generator().manual_seed(T), dtype=torch.int32)
    words = torch.full((guard + rows,), -7, dtype=torch.int32, device="cuda")
    row_of, offsets = torch.empty(T, dtype=torch.int32, device="cuda"), torch.empty(E + 1, dtype=torch.int32, device="cuda")
    buffers = [ids.cuda(), row_of, words[guard:], offsets]
    if route.scratch_bytes:
        buffers.append(torch.empty(route.scratch_bytes, dtype=torch.uint8, device="cuda"))
    torch.cuda.synchronize()
    _native.launch_raw(route.handle, torch.cuda.current_stream().cuda_stream, [b.data_ptr() for b in buffers])
    torch.cuda.synchronize()
    want = formulas.moe_route_ref(ids, E, 1, T)
    assert torch.equal(row_of.cpu(), want[0].view(-1)) and torch.equal(offsets.cpu(), want[2])
    assert torch.equal(words[guard:guard + T].cpu(), want[1])
    assert bool((words[:guard] == -7).all()), "words before entry_of were written"
    assert bool((words[guard + T:] == -1).all()), "a row without an entry was left out"


def test_threads_whose_sorts_need_different_shared_memory():
    """Three sorts of the same kernel, each above the 48 KB that a launch gets unasked, and a fourth of the two-launch
    form: one thread's smaller limit must not reach another's launch."""
    import threading

    shapes = [(32768, 1, 1024, 184320), (2048, 1, 330, 57032), (16384, 1, 1000, 164384), (40000, 1, 600, 76800)]
    routes = [moe.build_moe_route(T, k, E, block=1) for T, k, E, _ in shapes]
    assert [r.smem for r in routes] == [s[3] for s in shapes] and all(r.block == (1024, 1, 1) for r in routes)
    ids = [torch.randint(0, E, (T, k), dtype=torch.int32, device="cuda") for T, k, E, _ in shapes]
    torch.cuda.synchronize()
    errors, done = [], [0] * len(shapes)
    start = threading.Barrier(len(shapes))

    def work(n):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                start.wait()
                for _ in range(300):
                    _, entry_of, _ = routes[n](ids[n])
                torch.cuda.current_stream().synchronize()
                order = torch.sort(ids[n].flatten(), stable=True).indices
                assert torch.equal(entry_of.long(), order)
            done[n] += 1
        except Exception as exc:  # noqa: BLE001
            errors.append(exc)

    threads = [threading.Thread(target=work, args=(n,)) for n in range(len(shapes))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors and done == [1] * len(shapes), errors
