"""Host side of the cache-maintenance operators on CPU: workspaces that captured graphs may hold, and the
arguments of the rotary scalings at the edges of their ranges."""

from __future__ import annotations

from types import SimpleNamespace

import torch

from kvssd_b200 import ops

CPU = torch.device("cpu")


def test_a_replaced_workspace_is_kept_with_its_status(monkeypatch):
    """A captured graph holds a workspace's address: the tensor stays when a larger one takes its place,
    what it has flagged so far goes on in the new one, and what it flags later is still found."""
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    spaces = ops._Workspaces()
    stream, other = SimpleNamespace(cuda_stream=7), SimpleNamespace(cuda_stream=8)
    first = spaces.get(CPU, stream, 100)
    address = first.data_ptr()
    first[:4].view(torch.int32).fill_(2)
    del first
    big = spaces.get(CPU, stream, 3 << 20)
    assert big.numel() >= 3 << 20 and big[:4].view(torch.int32).item() == 2 and not big[4:].any()
    assert spaces.get(CPU, stream, 100) is big
    words = spaces.status_words(None, 7)
    assert len(words) == 2 and words[0] is big and words[1].data_ptr() == address
    spaces.get(CPU, other, 100)
    assert len(spaces.status_words(None, 7)) == 2 and len(spaces.status_words(None)) == 3
    assert spaces.status_words(0) == []
