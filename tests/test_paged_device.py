"""Calls made while another device is current: every entry point that looks at the device sees the
backend's.  Without a GPU: the library and the device switch are stand-ins."""

from __future__ import annotations

import contextlib

import pytest
import torch

from breezetoken_amd import backend as module
from breezetoken_amd.backend import HipBackend


class _Device:
    """Device 1, which every tensor here lies on."""

    index = 1

    def __eq__(self, other):
        return True

    __hash__ = None


class _Library:
    """Notes each entry point with the device that was current; paged workspaces by its CUs."""

    def __init__(self, seen, current):
        self.seen, self.current = seen, current

    def __getattr__(self, name):
        def call(*args):
            self.seen.append((name, self.current[0]))
            return 1024 * (1 + self.current[0]) if name.endswith("_bytes") else 0

        return call


@pytest.mark.parametrize("start", [0, 1])
def test_workspace_and_launch_see_the_backends_device(monkeypatch, start):
    current, seen = [start], []

    @contextlib.contextmanager
    def switched(dev):
        before, current[0] = current[0], dev.index
        yield
        current[0] = before

    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: current[0])
    monkeypatch.setattr(torch.cuda, "device", switched)
    monkeypatch.setattr(module, "_stream", lambda dev: 0)
    be = HipBackend.__new__(HipBackend)
    be._dev, be._lib = _Device(), _Library(seen, current)
    k = torch.zeros(4, 16, 2, 128, dtype=torch.bfloat16)
    table, lens = torch.zeros(2, 3, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    be.attention_paged(torch.zeros(2, 8, 128), k, k.clone(), table, lens, 1.0)
    assert seen == [("bt_paged_workspace_bytes", 1), ("bt_gqa_decode_paged", 1)] and current == [start]
