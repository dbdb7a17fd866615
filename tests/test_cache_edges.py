"""Host side of the cache-maintenance operators on CPU: workspaces that captured graphs may hold, and the
arguments of the rotary scalings at the edges of their ranges."""

from __future__ import annotations

import ctypes
import math
from types import SimpleNamespace

import pytest
import torch

from kvssd_b200 import RotaryEmbedding, _native, ops

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


def test_a_status_word_for_a_captured_call(monkeypatch):
    """A stream without a workspace borrows a word that no graph clears."""
    spaces = ops._Workspaces()
    capturing = True
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing)
    in_graph, eager = SimpleNamespace(cuda_stream=7), SimpleNamespace(cuda_stream=8)
    assert spaces.any_status_word(None) is None
    spaces.get(CPU, in_graph, 100)
    assert spaces.any_status_word(None) is None
    capturing = False
    buf = spaces.get(CPU, eager, 100)
    assert spaces.any_status_word(None) == buf.data_ptr() and spaces.any_status_word(0) is None


def weights_scratch(queries, places, qh, kvh, d, bits=4, group=32, bt=128):
    need = ctypes.c_size_t()
    _native.check(_native.library().kvssd_b200_attention_weights_scratch_size(
        queries, -(-places // bt), bt, qh, kvh, d, bits, group, ctypes.byref(need)), "scratch size")
    return need.value


@pytest.mark.parametrize("d, group, bt", [(128, 32, 128), (256, 16, 16), (80, 16, 128), (64, 64, 1)])
def test_weights_scratch_follows_what_is_used(d, group, bt):
    """8 bytes a part and query row. The parts of a row: no more than there are tiles (of 32 places, of 16
    for eight warps), and as many as come to 8 MB, or as four CTAs an SM shared by the KV heads, or as runs
    of 510 blocks (of whole tiles of 128 places)."""
    for kvh, places, queries in ((8, 131_072, 2048), (8, 1 << 20, 64), (1, 65_536, 32), (300, 5000, 3), (2, 40, 1)):
        rows = queries * kvh * 4
        parts, rest = divmod(weights_scratch(queries, places, 4 * kvh, kvh, d, group=group, bt=bt), 8 * rows)
        assert rest == 0 and parts >= 1
        blocks = -(-places // bt)
        run = 128 * max(1, 510 * bt // 128)
        assert parts <= max(1, 592 // kvh, (1 << 20) // rows, -(-blocks * bt // run))
        assert parts <= max(-(-blocks * bt // 32), -(-blocks * -(-bt // 16) // 8))


@pytest.mark.parametrize("kw, text", [
    (dict(base=math.nan), "base"), (dict(base=math.inf), "base"), (dict(scaling="linear", factor=math.nan), "factor"),
    (dict(scaling="yarn", factor=math.inf, original_length=64), "factor"),
    (dict(scaling="yarn", factor=2.0, original_length=64, high=math.inf), "finite"),
    (dict(scaling="smooth", factor=2.0, original_length=64, low=math.nan), "ascending"),
    (dict(scaling="smooth", factor=2.0, original_length=64, high=math.nan), "ascending")])
def test_rotary_embedding_refuses_what_is_no_number(kw, text):
    """They would make every frequency, and so every key, NaN without a word."""
    with pytest.raises(ValueError, match=text):
        RotaryEmbedding(128, **kw)
