"""CPU: the workspaces that the Python entry points keep."""
import weakref

import torch

from nvjsel import _tensors

CPU = torch.device("cpu")


def test_a_larger_call_keeps_the_workspace_that_a_graph_may_hold():
    """Calls captured before write to the address that they were captured with."""
    pool = _tensors._WorkspacePool()
    for kind in ("lm_head", "sample"):
        first = pool.get(CPU, 0, kind, 5000)
        held = weakref.ref(first)
        assert pool.get(CPU, 0, kind, 4000) is first
        del first
        larger = pool.get(CPU, 0, kind, 50000)
        assert held() is not None and larger.numel() >= 50000 and int(larger.sum()) == 0


def test_kept_workspaces_stay_few():
    """Growing a byte at a time holds less than four times what the largest call needs."""
    pool = _tensors._WorkspacePool()
    refs = []
    for n in range(5000, 6000):
        refs.append(weakref.ref(pool.get(CPU, 0, "sample", n)))
    held = {id(r()): r().numel() for r in refs if r() is not None}
    assert sum(held.values()) < 4 * 6000
