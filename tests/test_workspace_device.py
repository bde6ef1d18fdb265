"""A workspace's device may be given in every form that torch takes."""

from __future__ import annotations

import pytest

from ptxgen import attention


@pytest.mark.gpu
@pytest.mark.parametrize("form", [None, "cuda", "cuda:0", 0, "object", "object with index"])
def test_forms_of_a_device(cuda, form) -> None:
    import torch

    device = {"object": torch.device("cuda"), "object with index": torch.device("cuda", 0)}.get(
        form, form)
    ws = attention.Workspace(device)
    k = torch.randn((4, 1, 16, 64), device="cuda")
    table = torch.arange(4, dtype=torch.int32, device="cuda")[None]
    lens = torch.tensor([1], dtype=torch.int32, device="cuda")
    q = torch.randn((1, 2, 64), device="cuda")
    got = attention.decode(q, k, k, table, lens, workspace=ws)
    ws.check()
    # one key: its value, whatever the query (f32 products of two 11-bit parts: 2^-21 of it)
    assert float((got[0] - k[0, 0, 0]).abs().max()) <= 2.0 ** -20 * float(k.abs().max())


def test_a_device_with_an_index_is_the_buffer_s(monkeypatch) -> None:
    import torch

    from ptxgen.attention import Workspace

    zeros, asked = torch.zeros, []

    def host(n, dtype, device):
        asked.append(device)
        return zeros(1, dtype=dtype)

    monkeypatch.setattr(torch, "zeros", host)
    monkeypatch.setattr(attention, "wait_until_set", lambda device: asked.append(device))
    for device in (None, "cuda", torch.device("cuda:1")):
        asked.clear()
        w = Workspace(device)
        assert w.device == w.buffer.device == asked[1] and asked[0] == (device or "cuda")
