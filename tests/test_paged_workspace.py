"""The workspace of the paged attention calls is sized by the device that it lies on (no GPU needed)."""
import contextlib

import pytest
import torch


@pytest.mark.parametrize("current", [0, 1])
@pytest.mark.parametrize("device,want", [("cuda:0", 0), ("cuda:1", 1), ("cuda", None), (torch.device("cuda", 1), 1)])
def test_workspace_is_sized_by_its_device(monkeypatch, current, device, want):
    from vantablack_b200 import build
    build.build()
    from vantablack_b200 import ops
    now = [current]

    @contextlib.contextmanager
    def on(dev):
        before, now[0] = now[0], dev
        yield
        now[0] = before

    class Lib:  # a device of more SMs has larger workspaces
        @staticmethod
        def vtb_cuda_paged_attn_workspace_bytes(*_):
            return 1000 * (now[0] + 1)

    made = []
    monkeypatch.setattr(ops, "_current_device", lambda: now[0])
    monkeypatch.setattr(ops, "lib", Lib)
    monkeypatch.setattr(torch.cuda, "device", on)
    monkeypatch.setattr(torch, "empty", lambda n, dtype, device: made.append((n, dtype, torch.device(device))))
    ops._workspace_bytes.cache_clear()
    try:
        ops.paged_attention_workspace(torch.float16, 8, 2, 64, device=device)
    finally:
        ops._workspace_bytes.cache_clear()
    dev = current if want is None else want
    assert made == [(1000 * (dev + 1), torch.uint8, torch.device(device))] and now[0] == current
