"""Results of calls on a given stream come from that stream's memory. From the current stream's, a
block that the current stream still reads could be written at once, and a result that is dropped
early could be given away while the call still writes it."""

from __future__ import annotations

import pytest

from ptxgen import attention, logprob


def _stream_of(t) -> int:
    import torch

    at = t.data_ptr()
    for s in torch.cuda.memory_snapshot():
        if s["address"] <= at < s["address"] + s["total_size"]:
            return s["stream"]
    raise AssertionError("not the allocator's memory")


def _calls(stream):
    import torch

    def ints(*x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")

    g = torch.Generator(device="cuda").manual_seed(1)
    k = torch.randn((40, 2, 16, 64), device="cuda", generator=g)
    q = torch.randn((3, 4, 64), device="cuda", generator=g)
    table = torch.arange(39, dtype=torch.int32, device="cuda").view(3, 13)
    lens, starts, ws = ints(200, 1, 64), ints(0, 1, 2, 3), attention.Workspace()
    x = torch.randn((5, 1000), device="cuda", generator=g)
    t, ones = ints(1, 2, 3, 4, 5), torch.ones(5, device="cuda")
    torch.cuda.synchronize()
    yield attention.decode(q, k, k, table, lens, workspace=ws, stream=stream)
    yield attention.prompt(q, starts, k, k, table, lens, workspace=ws, stream=stream)
    r = logprob.logprobs(x, t, top=3, stream=stream)
    for part in (r.logp, r.entropy, r.norm, r.top_logp, r.top_ids):
        yield part
    yield logprob.logprobs_grad(x, t, r, ones, ones, stream=stream)
    torch.cuda.synchronize()


@pytest.mark.gpu
def test_results_belong_to_the_stream_of_the_call(cuda) -> None:
    import torch

    side = torch.cuda.Stream()
    want = list(_calls(None))
    assert [_stream_of(t) for t in want] == [0] * 8
    got = list(_calls(side.cuda_stream))
    assert [_stream_of(t) for t in got] == [side.cuda_stream] * 8
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert torch.cuda.current_stream() == torch.cuda.default_stream()
    with torch.cuda.stream(side):  # the default stream from another one
        got = list(_calls(0))
        assert [_stream_of(t) for t in got] == [0] * 8
        assert torch.cuda.current_stream() == side
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        # the current stream by its handle, and by default
        for handle in (side.cuda_stream, None):
            assert [_stream_of(t) for t in _calls(handle)] == [side.cuda_stream] * 8
