"""Calls at once with the workspaces that they get by themselves: on two streams, from two threads on one stream.
Every comparison is of bits: no call's result may depend on what ran beside it."""
import threading

import pytest
import torch

import bounded_ref as ref
from abridgekv_b200 import _lib, codestep, compaction, decode, prefill

pytestmark = pytest.mark.gpu
DEV = "cuda"
HKV, G, D, PAGE = 2, 2, 128, 16


class Job:
    """A paged cache with what the entries over it need."""

    def __init__(self, lens, seed, group=G):
        c = ref.Paged(lens, HKV, D, PAGE, 0, seed=seed)
        g = torch.Generator().manual_seed(seed)
        self.kv, self.bt, self.seq = c.kv.to(DEV), c.table.to(DEV), c.seq.to(DEV)
        self.q = torch.randn((len(lens), HKV * group, D), generator=g).bfloat16().to(DEV)
        self.w = torch.rand((len(lens), HKV, c.width * PAGE), generator=g).to(DEV)
        self.pages = (self.bt,), (self.seq,)

    def decode(self, stream=None):
        return decode.paged_decode([self.q], [self.kv], *self.pages, chunk_tokens=64, stream=stream)

    def weighted(self):
        w = self.w.clone()
        return decode.paged_decode_weighted([self.q], [self.kv], *self.pages, [w], chunk_tokens=64) + [w]

    def one_unit(self):
        w = torch.zeros((len(self.seq), 1, self.w.shape[2]), device=DEV)
        starts = torch.arange(len(self.seq) + 1, dtype=torch.int32, device=DEV)
        out, lse = codestep.paged_prefill_window(self.q, self.kv, self.bt, self.seq, starts, max_query_len=1,
                                                 num_kv_heads=HKV, window=None, return_lse=True)
        codestep.paged_prompt_weights(self.q, lse, self.kv, self.bt, self.seq, starts, w, max_query_len=1,
                                      num_kv_heads=HKV)
        return [out, lse, w]

    def evict(self):
        kv = self.kv.clone()
        e = compaction.evict_by_weight([kv], *self.pages, [self.w], budget=300, num_sinks=4, num_recent=8)
        return [kv.view(torch.int16), e.seq_lens[0], e.weights[0]]


def backward(seed):
    g = torch.Generator().manual_seed(seed)
    q, k, v, do = (torch.randn((1, h, 300, 64), generator=g).bfloat16().to(DEV) for h in (4, 2, 2, 4))
    out, lse = prefill.window_forward(q, k, v, window=70, num_sinks=2, return_lse=True)
    return lambda: list(prefill.window_backward(q, k, v, out, do, lse, window=70, num_sinks=2))


def equal(got, want):
    return all(torch.equal(a, b) for a, b in zip(got, want, strict=True))


def test_an_older_entry_on_a_side_stream_beside_new_ones_on_the_default_stream():
    a, b, bwd = Job([2000, 1500, 700], 1), Job([900, 1100], 2), backward(3)
    calls = [b.weighted, b.evict, bwd, b.one_unit]
    alone, decoded = [f() for f in calls], a.decode()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    for _ in range(10):
        beside = [a.decode(stream=s) for _ in range(12)]
        got = [f() for f in calls for _ in range(2)]
        beside += [a.decode(stream=s) for _ in range(12)]
        torch.cuda.synchronize()
        assert all(equal(x, decoded) for x in beside)
        assert all(equal(x, alone[i // 2]) for i, x in enumerate(got))


def test_two_threads_on_one_stream():
    jobs = [Job([900, 1100], 4), Job([1300, 650], 5)]
    calls = [[j.weighted, j.evict, backward(6 + i), j.one_unit] for i, j in enumerate(jobs)]
    alone = [[f() for f in fs] for fs in calls]
    torch.cuda.synchronize()
    start, wrong = threading.Barrier(2), []

    def work(fs, want):
        start.wait()
        got = [[f() for f in fs] for _ in range(20)]
        torch.cuda.synchronize()
        wrong.extend(i for r in got for i, x in enumerate(r) if not equal(x, want[i]))

    threads = [threading.Thread(target=work, args=a) for a in zip(calls, alone)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_a_windowed_layer_on_two_streams_and_in_a_graph():
    """The attention backend without a workspace of its own: layers at once on two streams, and a captured step that is
    replayed after eager calls have needed larger workspaces."""
    from types import SimpleNamespace

    from abridgekv_b200 import attention

    impl = attention.AbkvAttentionImpl(HKV * G, D, D ** -0.5, num_kv_heads=HKV, sliding_window=700, num_sinks=3)

    def layer(j):
        B = len(j.seq)
        starts = torch.arange(B + 1, dtype=torch.int32)
        md = attention.AbkvMetadataBuilder().build(0, SimpleNamespace(
            num_reqs=B, num_actual_tokens=B, query_start_loc=starts.to(DEV), query_start_loc_cpu=starts, seq_lens=j.seq,
            _seq_lens_cpu=j.seq.cpu(), block_table_tensor=j.bt, slot_mapping=torch.full((B,), -1, device=DEV),
            max_query_len=1, causal=True))
        new = torch.zeros((B, HKV, D), dtype=torch.bfloat16, device=DEV)
        out = torch.zeros((B, HKV * G * D), dtype=torch.bfloat16, device=DEV)
        return lambda: impl.forward(None, j.q.view(B, -1), new, new, j.kv, md, out)

    # enough (sequence, KV head) pairs for the split kernel, whose partial results lie in the workspace
    layers = [layer(Job([1500] * 150 + [20] * i, 11 + i)) for i in range(2)]
    alone = [f().clone() for f in layers]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in layers]
    for _ in range(10):
        got = []
        for f, s in zip(layers * 3, streams * 3):
            with torch.cuda.stream(s):
                got.append(f().clone())
        torch.cuda.synchronize()
        assert all(torch.equal(x, alone[i % 2]) for i, x in enumerate(got))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = layers[0]()
    big = Job([1500] * 400, 13)
    want = big.weighted()
    for _ in range(3):
        out.zero_()
        g.replay()
        assert equal(big.weighted(), want)
        torch.cuda.synchronize()
        assert torch.equal(out, alone[0])


def test_a_graph_with_a_workspace_that_grows_afterwards():
    """Older and newer entries captured with the caller's workspace, which eager calls then outgrow; memory of the old
    buffer's size is taken and filled between the replays."""
    from abridgekv_b200.workspace import Workspace

    j, big, ws = Job([900, 1100], 21), Job([1500] * 60, 22), Workspace(DEV, 1 << 18)
    w = torch.zeros_like(j.w)

    def step():
        return (decode.paged_decode([j.q], [j.kv], *j.pages, chunk_tokens=64, workspace=ws) +
                decode.paged_decode_weighted([j.q], [j.kv], *j.pages, [w], chunk_tokens=64, workspace=ws))

    want = [t.clone() for t in step()]
    want_w, size = w.clone(), ws.nbytes
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    bw = torch.zeros_like(big.w)
    decode.paged_decode_weighted([big.q], [big.kv], *big.pages, [bw], chunk_tokens=64, workspace=ws)
    assert ws.nbytes > size
    others = [torch.full((size,), 85, dtype=torch.uint8, device=DEV) for _ in range(4)]
    for _ in range(3):
        w.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert equal(got, want) and torch.equal(w, want_w)
        assert all((x == 85).all() for x in others)
    assert ws.read_error() == 0


def test_threads_whose_cluster_kernels_need_different_shared_memory(monkeypatch):
    """One sequence with accumulators (scores in shared memory) in one thread, one without in others, each on its own
    stream: they share the kernel, whose limit of shared memory is the process's.  The bare C calls, so that the
    threads meet inside them."""
    jobs = [Job([9000], 31, group=8), Job([200], 32, group=8)]
    w = torch.zeros_like(jobs[0].w)  # 73 KB of shared memory against 37
    calls = [lambda: decode.paged_decode_weighted([jobs[0].q], [jobs[0].kv], *jobs[0].pages, [w]),
             lambda: decode.paged_decode_window([jobs[1].q], [jobs[1].kv], *jobs[1].pages, window=100)]
    entry, args = _lib.lib().abkv_decode_window, []

    class Recorder:
        def __getattr__(self, name):
            return getattr(real, name) if name != "abkv_decode_window" else lambda *a: args.append(a) or entry(*a)

    real = _lib.lib()
    monkeypatch.setattr(_lib, "lib", Recorder)
    streams, keep = [], []
    for f in (calls[0], calls[1], calls[1], calls[1]):
        streams.append(torch.cuda.Stream())
        with torch.cuda.stream(streams[-1]):
            keep.append(f())
    torch.cuda.synchronize()
    start, status = threading.Barrier(4), [set() for _ in args]

    def work(i):
        start.wait()
        for k in range(20000):
            status[i].add(entry(*args[i]))
            if k % 500 == 499:
                streams[i].synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert status == [{0}] * 4
