"""CPU: every library call of the KDA functions runs with its tensors' device current."""

from __future__ import annotations

import contextlib
import re
from pathlib import Path

import torch

from axiom_amd import kda


def test_call_makes_the_device_current(monkeypatch):
    state = dict(current=0, seen=[])

    @contextlib.contextmanager
    def device(d):
        old, state["current"] = state["current"], d.index
        yield
        state["current"] = old

    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(kda, "_current_device", lambda: state["current"])
    monkeypatch.setattr(kda, "_stream", lambda d: 100 + d.index)

    def entry(stream, *args):
        state["seen"].append((state["current"], stream, args))
        return 7

    assert kda._call(entry, torch.device("cuda", 1), "x") == 7 and kda._call(entry, torch.device("cuda", 0), "y", "z") == 7
    assert state["seen"] == [(1, 101, ("x",)), (0, 100, ("y", "z"))] and state["current"] == 0


def test_no_library_call_goes_past_it():
    text = Path(kda.__file__).read_text()
    assert len(re.findall(r"\b_call\(", text)) > 10
    assert re.findall(r"(\S+)\(_stream\(", text) == ["entry", "entry"]   # in _call itself
