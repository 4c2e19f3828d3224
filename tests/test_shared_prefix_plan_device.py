"""A plan is divided for the GPU it is for, not for the current one: checked on the host with
stand-ins for the device calls."""

import types

import torch

from agentserve_b200 import _native as N
from agentserve_b200 import ops
from tests.test_shared_prefix_host import lib  # noqa: F401


def test_the_library_divides_for_the_plans_device(lib, monkeypatch):  # noqa: F811
    current, seen, zeros = [0], [], torch.zeros

    class Device:
        def __init__(self, device):
            self.index = torch.device(device).index

        def __enter__(self):
            current.append(self.index)

        def __exit__(self, *exc):
            current.pop()

    class Library:
        def __getattr__(self, name):
            def call(*args):
                seen.append((name, current[-1]))
                return getattr(lib, name)(*args)
            return call

    def on_the_host(*size, device=None, pin_memory=False, **kw):
        return zeros(*size, **kw)

    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(torch.cuda, "Event", lambda: types.SimpleNamespace(
        synchronize=lambda: None, record=lambda: None))
    monkeypatch.setattr(torch, "zeros", on_the_host)
    monkeypatch.setattr(N, "load", Library)
    plan = ops.shared_prefix_plan([[0, 1]], [4], [5, 6, 7], 32, 8, 64, torch.bfloat16, "cuda:3")
    plan.load([], [], [5, 6, 7])
    assert len(seen) == 4 and {device for _, device in seen} == {3}, seen
    assert current == [0]
