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

    class Stream:
        device_index = 0

    class Lib:
        @staticmethod
        def cottus_rope_append_decode_workspace_size(p):
            return 1 << 20

    monkeypatch.setattr(ops, "lib", lambda: Lib)
    monkeypatch.setattr(ops, "_require", lambda *a, **k: None)
    monkeypatch.setattr(ops, "make_step_params", lambda *a, **k: ops.DecodeStepParams())
    monkeypatch.setattr(torch.cuda, "stream", lambda stream: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    x, side = torch.zeros(1, 2, 64), Stream()
    with pytest.raises(KeyboardInterrupt):
        ops.rope_append_decode(x, x, x, x, x, x, x, num_kv_heads=2, head_dim=64, block_size=16, stream=side,
                               workspace_of=Batch())
    assert seen == [side]


CALLS = [("paged_decode", 4), ("lse_combine", 2), ("rope", 3), ("rope_append", 7), ("rope_append_decode", 7),
         ("qkv_rope_append", 6), ("o_proj_residual", 3), ("attention_block", 7), ("paged_gather", 3)]


@pytest.mark.parametrize("name, args", CALLS)
def test_a_stream_of_another_device_is_refused(monkeypatch, name, args):
    """Its kernels would run on that device with this one's addresses."""

    class Stream:
        device_index = 1

    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    with pytest.raises(ValueError, match="cuda:1.*cuda:0"):
        getattr(cb, name)(*[torch.zeros(1, 2, 64)] * args, stream=Stream())


@pytest.mark.parametrize("name, args", CALLS)
def test_calls_run_within_their_stream(monkeypatch, name, args):
    """Allocations of a call with a stream are served from that stream's memory."""
    inside, log = [], []

    class Stream:
        device_index = 0

    @contextlib.contextmanager
    def on(stream):
        inside.append(stream)
        yield
        inside.pop()

    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "stream", on)

    def stop(*a, **k):
        log.append(list(inside))
        raise KeyboardInterrupt

    monkeypatch.setattr(ops, "_require", stop)
    monkeypatch.setattr(ops, "qkv_rope_append", stop)
    monkeypatch.setattr(torch, "zeros", stop)
    side, x = Stream(), torch.ones(1, 2, 64)

    class Batch:
        num_blocks = 1

        def __len__(self):
            return 1

        positions = block_table = context_lens = x

        block_size = 16

    kw = dict(num_kv_heads=2, head_dim=64, block_size=16)
    if name == "attention_block":
        kw = dict(num_heads=2, num_kv_heads=2, head_dim=64)
    elif name == "qkv_rope_append":
        monkeypatch.undo()
        monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
        monkeypatch.setattr(torch.cuda, "stream", on)
        monkeypatch.setattr(ops, "_require", stop)
        kw["num_heads"] = 2
    elif name == "paged_gather":
        kw["max_context"] = 16
    elif name in ("lse_combine", "rope", "o_proj_residual"):
        kw = {}
    first = [Batch()] if name == "attention_block" else []
    with pytest.raises(KeyboardInterrupt):
        getattr(cb, name)(*first, *[x] * (args - len(first)), stream=side, **kw)
    assert log == [[side]]


def test_the_default_stream_of_another_device_is_refused():
    """Its handle is that of this device's default stream: the call would run, on the wrong one."""

    class Stream:
        device_index, cuda_stream = 1, 0

    assert ops._raw_stream(Stream(), 1) == 0
    with pytest.raises(ValueError, match="cuda:1.*cuda:0"):
        ops._raw_stream(Stream(), 0)
