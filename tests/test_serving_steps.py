"""What the token-by-token path decides on the host before anything reaches a GPU: which device a plan is made
for, steps that do not match the cache.  No GPU is needed; nothing here launches a kernel."""

from __future__ import annotations

import contextlib

import pytest
import torch

from ue5m3_fp4 import _native
from ue5m3_fp4.serving import operators


def test_attention_workspace_is_planned_on_the_operands_device(monkeypatch):
    """The plan depends on the device's number of SMs: it is asked for with that device current, and kept apart
    from another device's."""

    current, asked = [0], []

    class Library:
        @staticmethod
        def ue5m3_paged_attention_workspace_bytes(*sizes):
            asked.append(current[0])
            return 1000 * (current[0] + 1) + sizes[0]

    @contextlib.contextmanager
    def device(index):
        before, current[0] = current[0], index
        yield
        current[0] = before

    monkeypatch.setattr(_native, "load", Library)
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: current[0], raising=False)
    operators._workspace_bytes.cache_clear()
    try:
        assert operators._workspace_bytes(0, 5, 1) == 1005
        assert operators._workspace_bytes(1, 5, 1) == 2005
        current[0] = 1
        assert operators._workspace_bytes(0, 5, 1) == 1005 and operators._workspace_bytes(0, 6, 1) == 1006
        assert asked == [0, 1, 0] and current[0] == 1
    finally:
        operators._workspace_bytes.cache_clear()
