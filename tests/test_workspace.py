"""Which workspace a call gets, without a GPU: the streams and the capture state are faked, the buffers are host tensors."""
import gc
import threading
import weakref
from types import SimpleNamespace

import pytest
import torch

from abridgekv_b200 import workspace as W

DEV = torch.device("cuda", 0)


class Stream:
    """The current stream as the fakes see it."""
    raw, capturing = 0, False


@pytest.fixture
def now(monkeypatch):
    s = Stream()
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda i: s.raw, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_isCurrentStreamCapturing", lambda: s.capturing, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    real = W.Workspace.__init__
    monkeypatch.setattr(W.Workspace, "__init__", lambda self, device=None, *a, **kw: real(self, "cpu", *a, **kw))
    monkeypatch.setattr(W.Workspace, "on", property(lambda self: DEV), raising=False)
    monkeypatch.setattr(W, "_per_device", {})
    return s


def in_thread(fn):
    out = []
    t = threading.Thread(target=lambda: out.append(fn()))
    t.start()
    t.join()
    return out[0]


def test_a_call_shares_its_buffer_with_no_other_stream_thread_or_entry(now):
    first = W.call_workspace(DEV, 300)[0]
    assert W.call_workspace(DEV, 200)[0] is first and first.nbytes >= 300
    assert first is not W.default_workspace(DEV)  # which older entries take on any stream and inside captures
    other = in_thread(lambda: W.call_workspace(DEV, 300)[0])
    assert other is not first and W.call_workspace(DEV, 300)[0] is first
    now.raw = 77
    side, raw = W.call_workspace(DEV, 300)
    assert raw == 77 and side not in (first, other) and W.call_workspace(DEV, 300)[0] is side
    now.capturing = True
    graphs = [W.call_workspace(DEV, 300)[0] for _ in range(2)]
    assert graphs[0] is not graphs[1] and not {id(g) for g in graphs} & {id(first), id(other), id(side)}
    mine = W.Workspace(DEV, 256)
    assert W.call_workspace(DEV, 512, mine)[0] is mine and mine.nbytes == 512


def test_the_buffer_of_a_stream_can_be_found(now):
    first = W.call_workspace(DEV, 4096)[0]
    assert W.stream_workspace(DEV) is first and first.nbytes == 4096
    now.raw = 5
    assert W.stream_workspace(DEV) is W.call_workspace(DEV, 256)[0] is not first


@pytest.mark.parametrize("qlens", [[1, 1], [3, 2]])
def test_a_windowed_layer_leaves_the_choice_to_the_entries(monkeypatch, qlens):
    """The attention backend without a workspace hands none on: a shared one would meet another stream's calls."""
    from test_bounded_host import attention, codestep, decode, impl, metadata

    seen = []
    for mod, name in ((decode, "paged_decode_window"), (codestep, "paged_prefill_window")):
        monkeypatch.setattr(mod, name, lambda *a, **kw: seen.append(kw["workspace"]))
    monkeypatch.setattr(attention, "store_kv", lambda *a, **kw: None)
    monkeypatch.setattr(attention, "default_workspace", lambda device: W.Workspace("cpu"))
    T = sum(qlens)
    q, kv = torch.zeros(T, 1024, dtype=torch.bfloat16), torch.zeros(4, 2, 16, 2, 128, dtype=torch.bfloat16)
    new = torch.zeros(T, 256, dtype=torch.bfloat16)
    impl(sliding_window=32).forward(None, q, new, new, kv, metadata(qlens), q.clone())
    assert seen == [None]


def test_a_buffer_that_a_graph_uses_outlives_its_growth(now):
    ws = W.Workspace(DEV, 256)
    ws.ptr()
    ref = weakref.ref(ws._buf.untyped_storage())
    ws.ensure(512)
    gc.collect()
    assert ref() is None  # no graph: given back
    now.capturing = True
    at, storage = ws.ptr(), weakref.ref(ws._buf.untyped_storage())
    now.capturing = False
    ws._buf[0] = 4
    ws.ensure(4096)
    assert ws.ptr() != at and ws._buf[0] == 4 and ws.nbytes == 4096
    gc.collect()
    assert storage() is not None and [b.data_ptr() for b in ws._kept] == [at]
    ws.ensure(8192)  # the second buffer was in no graph
    assert [b.data_ptr() for b in ws._kept] == [at]


def test_a_captured_call_zeroes_its_header_alone(now, monkeypatch):
    """What is zeroed under capture is zeroed at every replay, scores of a hundred megabytes too."""
    sizes = []
    zero, zeros = torch.Tensor.zero_, torch.zeros
    monkeypatch.setattr(torch.Tensor, "zero_", lambda t: (sizes.append(t.numel()), zero(t))[1])
    monkeypatch.setattr(torch, "zeros", lambda n, **kw: (sizes.append(n), zeros(n, **kw))[1])
    now.capturing = True
    ws = W.call_workspace(DEV, 1 << 20)[0]
    assert sizes == [256] and ws.nbytes == 1 << 20 and not ws._buf[:256].any()
    now.capturing = False
    sizes.clear()
    assert not W.Workspace(DEV, 4096)._buf.any() and sizes == [4096]


def test_streams_and_workspaces_of_another_device_are_refused(now, monkeypatch):
    """Their kernels would run where the call's tensors are not."""
    monkeypatch.setattr(torch.cuda, "stream", lambda s: s)
    here, there = (SimpleNamespace(device=torch.device("cuda", i)) for i in (0, 1))
    assert W.call_scope(DEV, here) is here
    with pytest.raises(ValueError, match="stream"):
        W.call_scope(DEV, there)
    ws = W.Workspace()
    assert W.call_workspace(DEV, 256, ws)[0] is ws
    with pytest.raises(ValueError, match="workspace"):
        W.call_workspace(there.device, 256, ws)


def test_the_device_of_a_workspace():
    assert W.Workspace("cpu").on == torch.device("cpu")
