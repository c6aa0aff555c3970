"""Scratch buffers of the Python layer, on host memory: when a buffer is kept,
cleared and handed out again, and on which stream it is made."""
import contextlib

import pytest
import torch

cb = pytest.importorskip("cottus_b200")
from cottus_b200 import ops  # noqa: E402

CPU = torch.device("cpu")


@pytest.fixture(autouse=True)
def _own_cache(monkeypatch):
    monkeypatch.setattr(ops, "_WS", {})


@pytest.fixture
def capture(monkeypatch):
    state = {"on": False}
    monkeypatch.setattr(ops, "_capturing", lambda device: state["on"])
    return state


def test_a_buffer_is_kept_and_cleared_once(capture):
    a = ops.workspace(1000, CPU)
    assert a.numel() == 1 << 20 and not a.any()
    a[5] = 1
    assert ops.workspace(1 << 20, CPU).data_ptr() == a.data_ptr() and a[5] == 1
    assert ops.workspace(1000, CPU, "proj").data_ptr() != a.data_ptr()


def test_smaller_buffers_stay(capture):
    """A captured graph goes on using the buffer it was given."""
    a = ops.workspace(1 << 20, CPU)
    b = ops.workspace((1 << 20) + 1, CPU)
    assert b.numel() == 2 << 20 and not b.any() and b.data_ptr() != a.data_ptr()
    assert ops.workspace(10, CPU).data_ptr() == b.data_ptr()
    kept = [t.data_ptr() for t in ops._WS[("cpu", None, "decode")].buffers]
    assert kept == [a.data_ptr(), b.data_ptr()]


@pytest.mark.parametrize("kind", ["decode", "proj"])
def test_a_captured_buffer_serves_its_capture_alone(capture, kind):
    """What a capture makes is written at the first replay, not now: an eager call after it gets another one."""
    capture["on"] = True
    inside = ops.workspace(3 << 20, CPU, kind)
    capture["on"] = False
    outside = ops.workspace(3 << 20, CPU, kind)
    assert outside.data_ptr() != inside.data_ptr()
    capture["on"] = True
    assert ops.workspace(3 << 20, CPU, kind).data_ptr() == outside.data_ptr()  # one that exists serves captures too


def test_buffers_are_made_on_the_stream_that_uses_them(capture, monkeypatch):
    log = []

    @contextlib.contextmanager
    def on(stream):
        log.append(("enter", stream))
        yield
        log.append(("exit", stream))

    monkeypatch.setattr(torch.cuda, "stream", on)
    made = torch.zeros
    monkeypatch.setattr(torch, "zeros", lambda *a, **k: (log.append("zeros"), made(*a, **k))[1])
    ops.workspace(100, CPU, stream="side")
    assert log == [("enter", "side"), "zeros", ("exit", "side")]
    batch = cb.DecodeBatch(4, 16, 2, 2, device=CPU)
    del log[:]
    batch.workspace(5 << 20, "side")
    assert log == [("enter", "side"), "zeros", ("exit", "side")]


def test_a_batch_has_its_buffer_before_any_capture(capture):
    """Two layers of a step captured before the batch ever ran: one buffer, cleared when the batch was made."""
    batch = cb.DecodeBatch(4, 16, 2, 2, device=CPU)
    capture["on"] = True
    a, b = batch.workspace(2 << 20), batch.workspace(4 << 20)
    assert a.data_ptr() == b.data_ptr() and not a.any()
    assert batch.workspace(5 << 20).data_ptr() != a.data_ptr()


def test_fused_calls_take_the_workspace_on_their_stream(capture, monkeypatch):
    """rope_append_decode(stream=..., workspace_of=...) hands its stream on (a buffer cleared on another stream might be
    cleared under the kernel)."""
    seen = []

    class Batch:
        def workspace(self, nbytes, stream=None):
            seen.append(stream)
            raise KeyboardInterrupt  # (nothing is launched)

    class Lib:
        @staticmethod
        def cottus_rope_append_decode_workspace_size(p):
            return 1 << 20

    monkeypatch.setattr(ops, "lib", lambda: Lib)
    monkeypatch.setattr(ops, "_require", lambda *a, **k: None)
    monkeypatch.setattr(ops, "make_step_params", lambda *a, **k: ops.DecodeStepParams())
    x = torch.zeros(1, 2, 64)
    with pytest.raises(KeyboardInterrupt):
        ops.rope_append_decode(x, x, x, x, x, x, x, num_kv_heads=2, head_dim=64, block_size=16, stream="side",
                               workspace_of=Batch())
    assert seen == ["side"]
