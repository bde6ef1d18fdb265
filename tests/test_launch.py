"""The call of an operator, on a torch with and without its private names for the current device and
stream."""

from __future__ import annotations

import importlib

import pytest

PRIVATE = ("_cuda_getDevice", "_cuda_getCurrentRawStream")


@pytest.fixture(params=["private names", "public names"])
def launch(request, monkeypatch):
    import torch

    from ptxgen import launch

    with monkeypatch.context() as m:
        if request.param == "public names":
            for name in PRIVATE:
                m.delattr(torch._C, name, raising=False)
        importlib.reload(launch)
    yield launch
    importlib.reload(launch)


@pytest.mark.gpu
def test_calls_run_on_the_current_device_and_stream(cuda, launch) -> None:
    import torch

    got = []

    def fn(*args):
        got.append((torch.cuda.current_device(), args))
        return 0

    device, side = torch.device("cuda", 0), torch.cuda.Stream()
    launch.call(fn, device, None, 1, 2)
    launch.call(fn, device, 77, 3)
    with torch.cuda.stream(side):
        launch.call(fn, device, None)
    assert got == [(0, (1, 2, torch.cuda.default_stream().cuda_stream)), (0, (3, 77)),
                   (0, (side.cuda_stream,))]


def test_the_public_names_serve_where_the_private_ones_are_missing(monkeypatch) -> None:
    import torch

    from ptxgen import launch

    class Stream:
        def __init__(self, index):
            self.cuda_stream = 1000 + index

    with monkeypatch.context() as m:
        for name in PRIVATE:
            m.delattr(torch._C, name, raising=False)
        m.setattr(torch.cuda, "current_device", lambda: 2)
        m.setattr(torch.cuda, "current_stream", Stream)
        importlib.reload(launch)
        got = []
        launch.call(lambda *args: got.append(args) or 0, torch.device("cuda", 2), None, 5)
        launch.call(lambda *args: got.append(args) or 0, torch.device("cuda", 2), 9, 5)
        assert got == [(5, 1002), (5, 9)]
    importlib.reload(launch)
