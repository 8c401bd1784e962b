"""Host side of the bounded-cache operators without a GPU: the C entries refuse bad arguments before any launch,
their workspace queries, the Python entries' refusals, and the attention backend's dispatch under a window."""
import ctypes as C
from types import SimpleNamespace

import pytest
import torch

from abridgekv_b200 import _lib, attention, codestep, compaction, decode, prefill

INVALID, WORKSPACE, UNSUPPORTED = 1, 2, 3
FAKE = 1 << 20  # never dereferenced: validation fails first


def ptrs(*v):
    return _lib.ptr_array(list(v))


def i32(*v):
    return (C.c_int32 * len(v))(*v)


def i64(*v):
    return _lib.i64_array(list(v))


def run(entry, base, bad):
    args = {**base, **bad}
    return getattr(_lib.lib(), entry)(*args.values())


# Each base call is whole but for its missing workspace (a status of its own, checked behind the arguments).
DECODE = dict(q=ptrs(FAKE), kv=ptrs(FAKE), bt=ptrs(FAKE), strides=i64(8), lens=ptrs(FAKE), blocks=i64(64), out=ptrs(FAKE),
              layers=1, B=2, Hq=8, Hkv=2, D=128, page=16, pages=8, scale=0.1, chunk=0, windows=i32(32), sinks=i32(4),
              weights=ptrs(FAKE), wstrides=i64(256, 128), wrows=128, units=2, ws=0, nbytes=0, stream=None)


@pytest.mark.parametrize("bad,status", [
    ({}, WORKSPACE), (dict(ws=FAKE, nbytes=64), WORKSPACE), (dict(ws=FAKE + 8, nbytes=1 << 30), WORKSPACE),
    (dict(q=None), INVALID), (dict(lens=None), INVALID), (dict(out=None), INVALID), (dict(scale=0.0), INVALID),
    (dict(scale=float("nan")), INVALID), (dict(layers=0), INVALID), (dict(B=0), INVALID), (dict(windows=i32(-1)), INVALID),
    (dict(sinks=i32(-1)), INVALID), (dict(wstrides=None), INVALID), (dict(wrows=0), INVALID),
    (dict(units=4), INVALID), (dict(chunk=24), None), (dict(chunk=16384), None), (dict(D=96), UNSUPPORTED),
    (dict(Hkv=3, Hq=9, units=3), None), (dict(page=8), UNSUPPORTED), (dict(Hq=7), None), (dict(Hq=32), None),
    (dict(q=ptrs(FAKE + 4), ws=FAKE, nbytes=1 << 30), INVALID), (dict(q=ptrs(0), ws=FAKE, nbytes=1 << 30), INVALID),
    (dict(weights=ptrs(0), ws=FAKE, nbytes=1 << 30), INVALID), (dict(strides=i64(0), ws=FAKE, nbytes=1 << 30), INVALID),
    (dict(bt=ptrs(FAKE + 2), ws=FAKE, nbytes=1 << 30), INVALID), (dict(blocks=i64(0), ws=FAKE, nbytes=1 << 30), INVALID),
])
def test_decode_window_entry(bad, status):
    st = run("abkv_decode_window", DECODE, bad)
    assert st == status if status else st in (INVALID, UNSUPPORTED), st


def test_decode_window_workspace():
    size = _lib.lib().abkv_decode_window_workspace_size

    def n(layers=1, B=2, Hq=8, Hkv=2, D=128, page=16, pages=512, chunk=0, w=None, s=None, units=0):
        return size(layers, B, Hq, Hkv, D, page, pages, chunk, w, s, units)
    assert n() > 0 and n() % 256 == 0
    assert n(units=2) >= n() and n(units=1) >= n()
    assert n(w=i32(64), s=i32(4), chunk=64) <= n(chunk=64)  # a window needs no more partial results than the whole cache
    assert n(D=96) == n(B=0) == n(page=8) == n(Hq=9) == n(w=i32(-1)) == n(units=3) == n(layers=0) == 0
    # scores of every layer of a large call do not have to fit at once
    big = n(layers=36, B=64, Hq=32, Hkv=8, pages=2048, w=(C.c_int32 * 36)(), s=(C.c_int32 * 36)(), units=8)
    assert 0 < big < (2 << 30)


EVICT = dict(kv=ptrs(FAKE), bt=ptrs(FAKE), strides=i64(8), dst=None, dstrides=None, lens=ptrs(FAKE), new=ptrs(FAKE + 64),
             blocks=i64(64), w=ptrs(FAKE), ws_=i64(256, 128), wrows=128, wout=ptrs(FAKE), wouts=i64(256, 128), worows=128,
             keep=None, budgets=i32(64), layers=1, B=2, units=2, layout=0, Hkv=2, D=128, page=16, pages=8, sinks=4,
             recent=8, ws=0, nbytes=0, stream=None)


@pytest.mark.parametrize("bad,status", [
    ({}, WORKSPACE), (dict(ws=FAKE, nbytes=256), WORKSPACE), (dict(ws=FAKE + 64, nbytes=1 << 30), WORKSPACE),
    (dict(keep=ptrs(FAKE), ws=FAKE, nbytes=64), WORKSPACE), (dict(kv=None), INVALID), (dict(w=None), INVALID),
    (dict(wout=None), INVALID), (dict(budgets=None), INVALID), (dict(budgets=i32(0)), INVALID),
    (dict(budgets=i32(11)), INVALID), (dict(sinks=-1), INVALID), (dict(recent=-1), INVALID), (dict(units=3), INVALID),
    (dict(layout=2), INVALID), (dict(wrows=0), INVALID), (dict(page=0), INVALID), (dict(new=ptrs(FAKE)), INVALID),
    (dict(dst=ptrs(FAKE), dstrides=i64(4)), INVALID), (dict(dst=ptrs(FAKE + 4)), INVALID),
    (dict(dst=ptrs(FAKE + 4), dstrides=i64(0)), INVALID), (dict(kv=ptrs(FAKE + 8)), INVALID), (dict(keep=ptrs(0)), INVALID),
    (dict(D=96), UNSUPPORTED), (dict(Hkv=3, units=1), UNSUPPORTED), (dict(B=9000), UNSUPPORTED),
    (dict(pages=1 << 28), UNSUPPORTED), (dict(layers=0), INVALID), (dict(strides=i64(0)), INVALID),
    (dict(sinks=1 << 30, recent=1 << 30, budgets=i32(1 << 30)), INVALID),
])
def test_evict_entry(bad, status):
    assert run("abkv_evict_by_weight", EVICT, bad) == status


def test_evict_workspace():
    size = _lib.lib().abkv_evict_by_weight_workspace_size
    assert size(2, 3, 4, i32(100, 50)) >= 256 + 3 * 4 * 150 * 4
    assert size(0, 3, 4, i32(1)) == size(1, 0, 4, i32(1)) == size(1, 1, 0, i32(1)) == size(1, 1, 1, None) == 0
    assert size(2, 1, 1, i32(5, 0)) == 0


PROMPT = dict(q=FAKE, qr=1024, qh=128, out=FAKE, orow=1024, oh=128, lse=None, starts=FAKE, kv=FAKE, layout=0, blocks=64,
              page=16, bt=FAKE, stride=8, lens=FAKE, R=2, Hq=8, Hkv=2, D=128, mq=50, T=100, scale=0.1, window=32, sinks=4,
              ws=0, nbytes=0, stream=None)


@pytest.mark.parametrize("bad,status", [
    ({}, WORKSPACE), (dict(ws=FAKE, nbytes=16), WORKSPACE), (dict(ws=FAKE + 4, nbytes=256), WORKSPACE),
    (dict(q=None), INVALID), (dict(out=None), INVALID), (dict(starts=None), INVALID), (dict(kv=None), INVALID),
    (dict(bt=None), INVALID), (dict(lens=None), INVALID), (dict(mq=0), INVALID), (dict(window=-1), INVALID),
    (dict(sinks=-1), INVALID), (dict(scale=-1.0), INVALID), (dict(R=0), INVALID), (dict(T=0), INVALID),
    (dict(Hq=9), INVALID), (dict(layout=5), INVALID), (dict(D=64), UNSUPPORTED), (dict(page=24), UNSUPPORTED),
])
def test_paged_prefill_window_entry(bad, status):
    assert run("abkv_paged_prefill_window", PROMPT, bad) == status


WEIGHTS = dict(q=FAKE, qr=1024, qh=128, lse=FAKE, starts=FAKE, kv=FAKE, layout=0, blocks=64, page=16, bt=FAKE, stride=8,
               lens=FAKE, w=FAKE, wsb=256, wsu=128, wrows=128, units=2, R=2, Hq=8, Hkv=2, D=128, mq=50, rows=128, T=100,
               observe=0, scale=0.1, window=0, sinks=0, ws=0, nbytes=0, stream=None)


@pytest.mark.parametrize("bad,status", [
    ({}, WORKSPACE), (dict(ws=FAKE, nbytes=16), WORKSPACE), (dict(units=1, ws=FAKE, nbytes=256), WORKSPACE),
    (dict(q=None), INVALID), (dict(lse=None), INVALID), (dict(w=None), INVALID), (dict(units=4), INVALID),
    (dict(observe=-1), INVALID), (dict(window=-1), INVALID), (dict(mq=0), INVALID), (dict(mq=101), INVALID),
    (dict(rows=0), INVALID), (dict(wrows=0), INVALID), (dict(R=0), INVALID), (dict(Hq=9), INVALID),
    (dict(scale=0.0), INVALID), (dict(q=FAKE + 8), INVALID), (dict(kv=FAKE + 8), INVALID), (dict(layout=-1), INVALID),
    (dict(D=64), UNSUPPORTED), (dict(page=8), UNSUPPORTED), (dict(R=70000), UNSUPPORTED),
])
def test_prompt_weights_entry(bad, status):
    assert run("abkv_prompt_weights", WEIGHTS, bad) == status


def test_prompt_weights_workspace():
    size = _lib.lib().abkv_prompt_weights_workspace_size
    assert size(3, 8, 1000, 8) == 256 and size(3, 1, 1000, 1) == 256
    assert size(3, 8, 1000, 1) == 256 + 3 * 8 * 1000 * 4
    assert size(0, 8, 1000, 1) == size(3, 8, 0, 8) == size(3, 0, 10, 1) == 0


S3 = i64(8 * 64, 64, 8 * 64)
FORWARD = dict(q=FAKE, qs=S3, k=FAKE, ks=S3, v=FAKE, vs=S3, out=FAKE, os=S3, lo=None, lse=None, B=1, H=8, Hkv=2, S=100, D=64,
               scale=0.1, window=16, sinks=1, ws=0, nbytes=0, stream=None)
COMMON = [
    ({}, WORKSPACE), (dict(ws=FAKE, nbytes=64), WORKSPACE), (dict(ws=FAKE + 8, nbytes=1 << 30), WORKSPACE),
    (dict(q=None), INVALID), (dict(ks=None), INVALID), (dict(window=0), INVALID), (dict(window=-4), INVALID),
    (dict(sinks=-1), INVALID), (dict(S=0), INVALID), (dict(B=0), INVALID), (dict(H=9), INVALID), (dict(Hkv=0), INVALID),
    (dict(scale=-0.1), INVALID), (dict(q=FAKE + 2), INVALID), (dict(out=FAKE + 8), INVALID), (dict(lo=FAKE + 8), INVALID),
    (dict(D=96), UNSUPPORTED), (dict(H=256, Hkv=2), UNSUPPORTED), (dict(S=131073), UNSUPPORTED), (dict(B=70000), UNSUPPORTED),
]


@pytest.mark.parametrize("bad,status", COMMON)
def test_window_attention_entry(bad, status):
    assert run("abkv_window_attention", FORWARD, bad) == status


BACKWARD = dict(q=FAKE, qs=S3, k=FAKE, ks=S3, v=FAKE, vs=S3, out=FAKE, os=S3, lo=None, dout=FAKE, dos=S3, lse=FAKE, dq=FAKE,
                dqs=S3, dk=FAKE, dks=S3, dv=FAKE, dvs=S3, B=1, H=8, Hkv=2, S=100, D=64, scale=0.1, window=16, sinks=1, ws=0,
                nbytes=0, stream=None)


@pytest.mark.parametrize("bad,status", COMMON + [
    (dict(lse=None), INVALID), (dict(dout=None), INVALID), (dict(dq=None), INVALID), (dict(dv=FAKE + 8), INVALID),
    (dict(dqs=i64(8 * 64, 64, 8 * 64 + 4)), INVALID), (dict(dos=None), INVALID), (dict(B=65000, S=4130), UNSUPPORTED),
])
def test_window_attention_backward_entry(bad, status):
    assert run("abkv_window_attention_backward", BACKWARD, bad) == status


def test_window_attention_backward_workspace():
    size = _lib.lib().abkv_window_attention_backward_workspace_size
    assert size(2, 8, 333, 64) >= 2 * 8 * 333 * 4 and size(2, 8, 333, 64) % 256 == 0
    assert size(0, 8, 333, 64) == size(2, 0, 333, 64) == size(2, 8, 0, 64) == size(2, 8, 333, 96) == 0


# ---------------------------------------------------------------- Python entries: no CPU path
def test_python_entries_refuse_cpu_tensors():
    q, kv = torch.zeros(2, 8, 128, dtype=torch.bfloat16), torch.zeros(4, 2, 16, 2, 128, dtype=torch.bfloat16)
    bt, sl = torch.zeros(2, 2, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    qs, w = torch.tensor([0, 1, 2], dtype=torch.int32), torch.zeros(2, 2, 32)
    with pytest.raises(TypeError):
        decode.paged_decode_window([q], [kv], [bt], [sl], window=16)
    with pytest.raises(TypeError):
        decode.paged_decode_weighted([q], [kv], [bt], [sl], [w])
    with pytest.raises(TypeError):
        codestep.paged_prefill_window(q, kv, bt, sl, qs, max_query_len=1, num_kv_heads=2, window=16)
    with pytest.raises(TypeError):
        codestep.paged_prompt_weights(q, torch.zeros(2, 8), kv, bt, sl, qs, w, max_query_len=1, num_kv_heads=2)
    with pytest.raises(TypeError):
        compaction.evict_by_weight([kv], [bt], [sl], [w], budget=16)
    with pytest.raises((TypeError, ValueError)):
        prefill.window_attention(*(torch.zeros(1, 2, 8, 64, dtype=torch.bfloat16) for _ in range(3)), window=4)


@pytest.mark.parametrize("window,sinks", [(-1, 0), (1 << 31, 0), (4, -1), (4, 1 << 31)])
def test_python_windows_out_of_range(window, sinks):
    with pytest.raises(ValueError):
        codestep._window(window, sinks)


def test_layout_of_a_cache():
    at = codestep._given_layout
    assert at(torch.zeros(5, 2, 16, 2, 64), None) == 0 and at(torch.zeros(2, 5, 16, 2, 64), None) == 1
    two = torch.zeros(2, 2, 16, 2, 64)
    with pytest.raises(ValueError, match="kv_layout"):  # either layout: not to be guessed
        at(two, None)
    assert at(two, 0) == 0 and at(two, 1) == 1
    for shape, layout in (((5, 2, 16, 2, 64), 1), ((2, 5, 16, 2, 64), 0), ((3, 4, 16, 2, 64), None), ((2, 2, 16, 64), 0),
                          ((2, 2, 16, 2, 64), 2)):
        with pytest.raises(ValueError):
            at(torch.zeros(shape), layout)


# ---------------------------------------------------------------- the attention backend under a window
def impl(**kw):
    return attention.AbkvAttentionImpl(8, 128, 0.1, num_kv_heads=2, **kw)


def metadata(qlens, causal=True):
    starts = torch.tensor([0] + list(torch.tensor(qlens).cumsum(0)), dtype=torch.int32)
    cm = SimpleNamespace(num_reqs=len(qlens), num_actual_tokens=sum(qlens), query_start_loc=starts,
                         query_start_loc_cpu=starts, seq_lens=torch.tensor([40] * len(qlens), dtype=torch.int32),
                         _seq_lens_cpu=torch.tensor([40] * len(qlens), dtype=torch.int32),
                         block_table_tensor=torch.zeros((len(qlens), 4), dtype=torch.int32),
                         slot_mapping=torch.zeros(sum(qlens), dtype=torch.int64), max_query_len=max(qlens), causal=causal)
    return attention.AbkvMetadataBuilder().build(0, cm)


@pytest.mark.parametrize("qlens,name", [([1, 1, 1], "paged_decode_window"), ([1, 5, 2], "paged_prefill_window")])
def test_backend_dispatches_a_window(monkeypatch, qlens, name):
    calls = []
    for mod, n in ((decode, "paged_decode"), (decode, "paged_decode_window"), (codestep, "paged_prefill"),
                   (codestep, "paged_prefill_window")):
        monkeypatch.setattr(mod, n, lambda *a, _n=n, **kw: calls.append((_n, kw)))
    T = sum(qlens)
    q, out = torch.zeros(T, 1024, dtype=torch.bfloat16), torch.zeros(T, 1024, dtype=torch.bfloat16)
    kv = torch.zeros(4, 2, 16, 2, 128, dtype=torch.bfloat16)
    ws = object()
    impl(sliding_window=32, num_sinks=4, workspace=ws).forward(None, q, None, None, kv, metadata(qlens), out)
    (called, kw), = calls
    assert called == name and kw["window"] == 32 and kw["num_sinks"] == 4 and kw["workspace"] is ws
    calls.clear()
    impl(sliding_window=-1, workspace=ws).forward(None, q, None, None, kv, metadata(qlens), out)
    assert calls[0][0] == name.removesuffix("_window") and "window" not in calls[0][1]


def test_backend_refuses_what_a_window_does_not_serve():
    for bad in (dict(sliding_window=0), dict(sliding_window=-2), dict(num_sinks=4), dict(sliding_window=8, num_sinks=-1)):
        with pytest.raises(ValueError):
            impl(**bad)
    q = torch.zeros(4, 1024, dtype=torch.bfloat16)
    kv = torch.zeros(4, 2, 16, 2, 128, dtype=torch.bfloat16)
    with pytest.raises(NotImplementedError, match="code step"):
        impl(sliding_window=8, workspace=object()).forward(None, q, None, None, kv, metadata([4], causal=False), q.clone())
    car = attention.CompressedKVSidecar.__new__(attention.CompressedKVSidecar)
    car.active_request_ids = ("a",)
    with pytest.raises(NotImplementedError, match="sliding window"):
        car.override_attention(layer_index=0, layer=SimpleNamespace(impl=impl(sliding_window=8)), query=q, kv_cache=kv,
                               attn_metadata=None, output=q)
