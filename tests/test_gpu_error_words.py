"""Device errors of operators that bring their own workspace, met by eager calls and by replays of captured graphs."""

from __future__ import annotations

import subprocess
import sys
from pathlib import Path

import pytest
import torch

from kairo_b200 import _lib, ops
from tests.test_gpu_gated import case

pytestmark = pytest.mark.gpu
BAD = _lib.DEVERR_BAD_INDEX


def graph_of(call, stream):
    stream.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        call()
    return g


def weights():
    x, dh, gate, up, wg, wu = case(40, 96, 128, 32, torch.bfloat16, keep=0.9)
    w = ops.gated_weights(gate, up)
    return x, w, w.entries[1].clone()


def test_a_replay_reports_to_the_stream_that_asks():
    x, w, kept = weights()
    ops.sparse_gated_linear(x, w, check=True)
    ops.pending_device_error()
    g = graph_of(lambda: ops.sparse_gated_linear(x, w), torch.cuda.Stream())
    g.replay()
    assert ops.pending_device_error() == 0
    w.entries[1, 0] = 1 << 20
    g.replay()
    assert ops.pending_device_error() & 0xFF == BAD
    assert ops.pending_device_error() == 0
    w.entries[1] = kept
    g.replay()
    assert ops.pending_device_error() == 0


def test_replays_leave_other_errors():
    """A word first met in a capture reads 0 before the first replay, and a replay wipes nothing that eager calls recorded."""
    x, w, kept = weights()
    s = torch.cuda.Stream()
    g = graph_of(lambda: ops.sparse_gated_linear(x, w), s)
    with torch.cuda.stream(s):
        assert ops.pending_device_error() == 0
        ops.sparse_gated_linear(x, w, check=True)
        w.entries[1, 0] = -1
        ops.sparse_gated_linear(x, w)
        w.entries[1] = kept
        g.replay()
        assert ops.pending_device_error() & 0xFF == BAD
        assert ops.pending_device_error() == 0


def test_more_streams_than_words():
    """Words are handed out until they run out; the last one then serves several streams."""
    index = torch.cuda.current_device()
    kept = dict(_lib._error_words)
    try:
        at = {_lib._error_word_of(index, 10**12 + i).data_ptr() for i in range(2000)}
        assert 100 < len(at) < 2000 and all(a % 256 == 0 for a in at)
        assert not at & {w.data_ptr() for k, w in kept.items() if k[0] == index}
    finally:
        _lib._error_words.clear()
        _lib._error_words.update(kept)


def test_every_word_is_read_at_once():
    """An error in the workspace of the stream and one in its word: the first is told, both are cleared."""
    x, w, kept = weights()
    a = case(40, 96, 128, 32, torch.bfloat16, keep=0.9)[2]
    a.col_idx[1] = 1 << 20
    w.entries[1, 0] = 1 << 20
    ops.sparse_linear(x, a)
    ops.sparse_gated_linear(x, w)
    assert ops.pending_device_error(clear=False) & 0xFF == BAD
    assert ops.pending_device_error() & 0xFF == BAD
    assert ops.pending_device_error() == 0


FIRST = """
import torch
from kairo_b200 import ops
x, w = torch.randn(40, 64, device="cuda").bfloat16(), torch.randn(300, 64, device="cuda").bfloat16()
ids = torch.randint(0, 300, (40,), device="cuda")
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    loss, lse = ops.linear_cross_entropy(x, w, ids, return_lse=True)
assert ops.pending_device_error() == 0
g.replay()
assert ops.pending_device_error() == 0
assert torch.equal(loss, ops.linear_cross_entropy(x, w, ids, check=True))
print("same")
"""


def test_first_call_of_a_process_in_a_capture():
    run = subprocess.run([sys.executable, "-c", FIRST], cwd=Path(__file__).resolve().parent.parent, capture_output=True,
                         text=True, timeout=300)
    assert run.returncode == 0 and run.stdout.strip() == "same", run.stderr[-2000:]
