"""Selections of two threads on one stream, which share a workspace: the order in which their
launches reach the stream, on the CPU, and the results of many calls that two threads queue
without waiting for any, on the GPU."""
import threading

import pytest
import torch

import nvjsel
from tests.launch_recorder import launches

SELECT = """('nvjsel_beam_select', [P, I, I, I, I, L, L, P, P, I, I, P, P, P, P, Z, P],
 [0x1000, 1, {0}, {1}, {2}, {1} * {2}, {2}, 0x1000, None, 0, 8, 0x1000, 0x1000, 0x1000, 0x1000, 1 << 40, None])"""


def test_no_call_comes_between_a_scan_and_its_join(tmp_path):
    order = launches(tmp_path, SELECT.format(24, 8, 20011), SELECT.format(2, 4, 9001))
    assert [thread for thread, _ in order] == ["first", "first", "other"]
    for (_, name), part in zip(order, ("beam_scan_kernel", "beam_join_kernel", "beam_select_kernel")):
        assert part in name


@pytest.mark.gpu
def test_two_threads_queue_small_and_large_selections():
    g = torch.Generator().manual_seed(3)
    shapes = [(2, 4, 9001), (24, 8, 20011)]  # of one launch, and of two
    data = [((torch.randn(b, w, v, generator=g) * 2).to(torch.bfloat16).cuda(), torch.randn(b, w, generator=g).cuda())
            for b, w, v in shapes]
    want = [nvjsel.beam_search_select(*x, num_candidates=8) for x in data]
    torch.cuda.synchronize()
    got = [[], []]
    start = threading.Barrier(2)

    def queue(at):
        start.wait()
        for _ in range(100):
            got[at].append(nvjsel.beam_search_select(*data[at], num_candidates=8))

    threads = [threading.Thread(target=queue, args=(at,)) for at in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for at in range(2):
        assert len(got[at]) == 100
        assert all(torch.equal(a, b) for out in got[at] for a, b in zip(out, want[at]))
