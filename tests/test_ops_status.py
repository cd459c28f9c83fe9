"""check_status against a stand-in for the device's word: what a call finds while the check clears what
it has reported belongs to the next check."""
import pytest
import torch

from yue2_rs_b200 import Yue2Error, ops


class Word:
    """An int32 of which the device sets a bit right after the check has read it."""

    def __init__(self, value, later):
        self.value, self.later = torch.tensor([value], dtype=torch.int32), later

    def item(self):
        bits = int(self.value.item())
        self.value |= self.later
        self.later = 0
        return bits

    def __getattr__(self, name):
        return getattr(self.value, name)


def test_bits_that_arrive_during_a_check_are_kept(monkeypatch):
    monkeypatch.setattr(torch.cuda, "synchronize", lambda device=None: None)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(ops, "_status", {0: (0, Word(1, 2))})
    device = torch.device("cuda", 0)
    with pytest.raises(Yue2Error, match="page index"):
        ops.check_status(device)
    with pytest.raises(Yue2Error, match="out of range"):
        ops.check_status(device)
    ops.check_status(device)
