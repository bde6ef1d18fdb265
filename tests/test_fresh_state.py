"""A cache or workspace that has just been made serves any stream: its zeros are there before the
first call on another stream reads them."""

from __future__ import annotations

import pytest

from ptxgen import attention
from ptxgen.cache import PagedCache


def _ints(*x):
    import torch

    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.gpu
def test_a_new_cache_and_workspace_on_another_stream(cuda) -> None:
    """They are made behind 50 ms of other work on the stream that makes them."""
    import torch

    making, calling = torch.cuda.Stream(), torch.cuda.Stream()
    slot, starts = _ints(1), _ints(0, 3000)
    g = torch.Generator(device="cuda").manual_seed(0)
    k, v = (torch.randn((3000, 1, 64), device="cuda", generator=g) for _ in range(2))
    q = torch.randn((1, 4, 64), device="cuda", generator=g)
    # what the allocator gives next is full of ones
    for s in (making, calling):
        with torch.cuda.stream(s):
            junk = [torch.full((n,), -1, dtype=torch.int32, device="cuda")
                    for n in (attention.WORKSPACE_BYTES // 4, 1, 2, 400, 1000, 2000)]
    del junk
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        with torch.cuda.stream(making):
            torch.cuda._sleep(100_000_000)
            c = PagedCache.allocate(1, 200, 1, 16, 64, 2, 200, dtype=torch.float32)
            torch.cuda._sleep(100_000_000)
            ws = attention.Workspace()
        s = calling.cuda_stream
        c.extend(slot, starts, stream=s)
        c.write(0, slot, starts, k, v, stream=s)
        got.append(attention.decode(q, c.k[0], c.v[0], c.table, c.lens, slots=slot, workspace=ws,
                                    stream=s))
        c.check()
        ws.check()
    p = torch.softmax(torch.einsum("qhd,kd->hk", q.double(), k[:, 0].double()) / 8, -1)
    want = p @ v[:, 0].double()
    for o in got:  # see tests/test_attention.py for the bound
        assert float((o[0].double() - want).abs().max()) <= 4e-5 * float(v.abs().max())


@pytest.mark.gpu
def test_a_workspace_may_be_made_under_capture(cuda) -> None:
    import torch

    k = torch.randn((4, 1, 16, 64), device="cuda")
    q, table, lens = torch.randn((1, 2, 64), device="cuda"), _ints(0, 1, 2, 3)[None], _ints(60)
    want = attention.decode(q, k, k, table, lens, workspace=attention.Workspace())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = attention.decode(q, k, k, table, lens, workspace=attention.Workspace())
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)


def test_the_wait_is_on_the_stream_that_set_it(monkeypatch) -> None:
    import torch

    from ptxgen import launch

    waits = []

    class Stream:
        def __init__(self, device):
            self.device = device

        def synchronize(self):
            waits.append(self.device)

    monkeypatch.setattr(torch.cuda, "current_stream", Stream)
    for capturing, want in ((False, ["cuda:1"]), (True, [])):
        monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing)
        waits.clear()
        launch.wait_until_set("cuda:1")
        assert waits == want
