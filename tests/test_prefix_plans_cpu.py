"""Plans of attention over a shared prefix around captures, and the division of the work (no GPU)."""
import contextlib

import pytest
import torch

from ds41rt_b200.models.base import RowsEngine


class Rows(RowsEngine):
    """An engine whose last rows were a prompt's, so that its plan is made when a pass asks for it."""

    def __init__(self):
        self.log, self.capturing, self.undescribed = [], False, True
        self.in_tokens = self.row_pos = self.row_slot = torch.zeros(4, dtype=torch.int32)
        self.long = True                                     # the first pass takes the form without a plan

    def settle(self):
        if self.undescribed:
            self.log.append("plan in capture" if self.capturing else "plan")
            self.undescribed = False

    def forward(self):
        if not self.long:
            self.settle()
        self.long = False
        self.log.append("captured" if self.capturing else "eager")


def test_plans_are_made_before_a_capture(monkeypatch):
    e = Rows()

    @contextlib.contextmanager
    def graph(g):
        e.capturing = True
        yield
        e.capturing = False

    monkeypatch.setattr(torch.cuda, "synchronize", lambda: None)
    monkeypatch.setattr(torch.cuda, "CUDAGraph", object)
    monkeypatch.setattr(torch.cuda, "graph", graph)
    e.capture(e.forward)
    assert e.log == ["plan", "eager", "captured"]
