"""The profiling harness's clock warm-up (no GPU needed): its launches are in the traced
averages, so they go through all sets of buffers as the others do."""

import os
import sys

import torch

_REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(_REPO, "flash-attention-cuda_amd", "profile"))

import profile_workload as pw  # noqa: E402


def test_the_warm_up_takes_every_set_in_turn(monkeypatch):
    monkeypatch.setattr(torch.cuda, "synchronize", lambda: None)
    calls = []
    pw._clock_warmup([lambda i=i: calls.append(i) for i in range(3)], seconds=0.01)
    assert len(calls) >= 10
    assert calls == [i % 3 for i in range(len(calls))]
