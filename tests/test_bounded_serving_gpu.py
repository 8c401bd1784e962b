"""The bounded-cache operators run together, as a server would: a prompt, its attention weights, eviction to a
budget, decode steps that go on accumulating, further evictions -- and windowed layers through the attention
backend.  Against a 64-bit restatement that keeps the rows of every (sequence, KV head) in lists.

Tolerances: outputs as in bounded_ref.  An accumulator is a sum of at most 100 weights, each within 2^-12 of
itself, added in 32 bits (half a step, 2^-24, of the sum per addition): 2^-12 + 100 x 2^-24 < 2^-11 of the sum.
Which rows an eviction keeps is compared exactly, against the selection from the accumulators it was given."""
from types import SimpleNamespace

import numpy as np
import pytest
import torch

import bounded_ref as ref
from abridgekv_b200 import attention, codestep, compaction, decode
from abridgekv_b200.workspace import Workspace

pytestmark = pytest.mark.gpu
DEV = "cuda"
HKV, G, D, PAGE = 2, 2, 128, 16
SCALE = D ** -0.5


class Rows:
    """One sequence in 64 bits: per KV head, the K and V rows that are left and their accumulated weights."""

    def __init__(self):
        self.k = [torch.zeros(0, D).double() for _ in range(HKV)]
        self.v = [torch.zeros(0, D).double() for _ in range(HKV)]
        self.w = [torch.zeros(0).double() for _ in range(HKV)]

    def append(self, k, v):  # [n, HKV, D]
        for h in range(HKV):
            self.k[h] = torch.cat([self.k[h], k[:, h].double()])
            self.v[h] = torch.cat([self.v[h], v[:, h].double()])
            self.w[h] = torch.cat([self.w[h], torch.zeros(len(k)).double()])

    def attend(self, q, pos, window=0, sinks=0, count=None):
        """q [m, HKV * G, D] at positions pos; the weights of the last `count` rows are added -> out, A."""
        outs, As = [], []
        for h in range(HKV):
            vis = ref.visible(pos, len(self.k[h]), window, sinks)
            o, A, _, p = ref.attend(q[:, h * G:(h + 1) * G], self.k[h], self.v[h], vis, SCALE)
            outs.append(o)
            As.append(A)
            if count is not None:
                self.w[h] = self.w[h] + p[len(q) - count:].sum((0, 1))
        return torch.cat(outs, 1), torch.cat(As, 1)

    def keep(self, h, rows):
        self.k[h], self.v[h], self.w[h] = self.k[h][rows], self.v[h][rows], self.w[h][rows]


def bf16(*shape, g):
    return torch.randn(shape, generator=g).bfloat16()


def check_acc(acc, seqs, tag):
    for b, s in enumerate(seqs):
        for h in range(HKV):
            got, want = acc[b, h].double().cpu(), s.w[h]
            n = len(want)
            assert (got[:n] - want).abs().le(2.0 ** -11 * want + 2.0 ** -40).all(), (tag, b, h)
            assert (got[n:] == 0).all(), (tag, b, h)


@pytest.mark.parametrize("graph", [False, True])
def test_prompt_evict_decode(graph):
    g = torch.Generator().manual_seed(7)
    lens, budget, sinks, recent, observe = [150, 41, 97], 64, 4, 8, 16
    B, width = len(lens), 12
    nb = B * width + 1
    kv = torch.full((nb, 2, PAGE, HKV, D), float("nan"), dtype=torch.bfloat16, device=DEV)
    bt = (torch.randperm(nb - 1, generator=g)[:B * width] + 1).view(B, width).int().to(DEV)
    seq = torch.tensor(lens, dtype=torch.int32, device=DEV)
    acc = torch.zeros((B, HKV, width * PAGE), device=DEV)
    seqs = [Rows() for _ in lens]
    ws = Workspace(DEV, 8 << 20)

    def slots(b, pos):
        return bt[b, pos // PAGE].long() * PAGE + pos % PAGE

    # prompt
    T = sum(lens)
    starts = torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32, device=DEV)
    q, k, v = bf16(T, HKV * G, D, g=g), bf16(T, HKV, D, g=g), bf16(T, HKV, D, g=g)
    sm = torch.cat([slots(b, torch.arange(n, device=DEV)) for b, n in enumerate(lens)])
    qd = q.to(DEV)
    attention.store_kv(k.to(DEV), v.to(DEV), kv, sm, workspace=ws)
    out, lse = codestep.paged_prefill_window(qd, kv, bt, seq, starts, max_query_len=max(lens), num_kv_heads=HKV, window=None,
                                             return_lse=True, workspace=ws)
    codestep.paged_prompt_weights(qd, lse, kv, bt, seq, starts, acc, max_query_len=max(lens), num_kv_heads=HKV,
                                  observe=observe, workspace=ws)
    at = 0
    for b, n in enumerate(lens):
        seqs[b].append(k[at:at + n], v[at:at + n])
        o, A = seqs[b].attend(q[at:at + n], list(range(n)), count=min(observe, n))
        ref.check_out(out[at:at + n], o, A, ("prompt", b))
        at += n
    check_acc(acc, seqs, "prompt")

    def evict(tag):
        before, old = acc.cpu().numpy(), seq.tolist()
        e = compaction.evict_by_weight([kv], [bt], [seq], [acc], budget=budget, num_sinks=sinks, num_recent=recent,
                                       return_keep=True, in_place_weights=True, workspace=ws)
        assert e.weights[0] is acc
        seq.copy_(e.seq_lens[0])
        for b, n in enumerate(old):
            assert int(seq[b]) == min(n, budget)
            for h in range(HKV):
                rows = ref.evict_rows(before[b, h], n, budget, sinks, recent)
                got = e.keep[0][b, h].cpu().numpy()
                assert (got[:len(rows)] == rows).all() and (got[len(rows):] == -1).all(), (tag, b, h)
                seqs[b].keep(h, rows)
        check_acc(acc, seqs, tag)

    evict("prompt")

    # decode: write the row, attend, accumulate; back to the budget whenever the longest has grown by 20
    sq = torch.zeros((B, HKV * G, D), dtype=torch.bfloat16, device=DEV)
    sk, sv = (torch.zeros((B, HKV, D), dtype=torch.bfloat16, device=DEV) for _ in range(2))
    so = torch.zeros_like(sq)
    rows = torch.arange(B, device=DEV)

    def step():
        pos = seq.long()
        attention.store_kv(sk, sv, kv, bt[rows, pos // PAGE].long() * PAGE + pos % PAGE, workspace=ws)
        seq.add_(1)
        decode.paged_decode_weighted([sq], [kv], [bt], [seq], [acc], outputs=[so], workspace=ws)

    cg = None
    if graph:
        keep = [t.clone() for t in (kv, seq, acc)]
        step()  # warm-up, taken back
        for t, s in zip((kv, seq, acc), keep):
            t.copy_(s)
        torch.cuda.synchronize()
        cg = torch.cuda.CUDAGraph()
        with torch.cuda.graph(cg):
            step()
    for i in range(50):
        q, k, v = bf16(B, HKV * G, D, g=g), bf16(B, HKV, D, g=g), bf16(B, HKV, D, g=g)
        sq.copy_(q)
        sk.copy_(k)
        sv.copy_(v)
        cg.replay() if graph else step()
        for b in range(B):
            seqs[b].append(k[b:b + 1], v[b:b + 1])
            o, A = seqs[b].attend(q[b:b + 1], [len(seqs[b].k[0]) - 1], count=1)
            ref.check_out(so[b:b + 1], o, A, ("step", i, b))
        if max(len(s.k[0]) for s in seqs) >= budget + 20:
            check_acc(acc, seqs, i)
            evict(i)
    check_acc(acc, seqs, "end")
    assert ws.read_error() == 0


def test_backend_with_a_window():
    """A windowed layer through the attention backend: a chunk of prompt rows, the rest of it, decode steps."""
    g = torch.Generator().manual_seed(11)
    window, sinks, width, B = 48, 4, 14, 2
    impl = attention.AbkvAttentionImpl(HKV * G, D, SCALE, num_kv_heads=HKV, sliding_window=window, num_sinks=sinks,
                                       workspace=Workspace(DEV, 8 << 20))
    kv = torch.full((B * width + 1, 2, PAGE, HKV, D), float("nan"), dtype=torch.bfloat16, device=DEV)
    bt = (torch.randperm(B * width, generator=g) + 1).view(B, width).int()
    seqs, done = [Rows() for _ in range(B)], [0] * B

    def step(qlens):
        T = sum(qlens)
        q, k, v = bf16(T, HKV * G, D, g=g), bf16(T, HKV, D, g=g), bf16(T, HKV, D, g=g)
        starts = torch.tensor([0] + list(np.cumsum(qlens)), dtype=torch.int32)
        sm = torch.cat([bt[b, (p := torch.arange(done[b], done[b] + n)) // PAGE].long() * PAGE + p % PAGE
                        for b, n in enumerate(qlens)])
        now = torch.tensor([d + n for d, n in zip(done, qlens)], dtype=torch.int32)
        # pages that the window has left behind are freed: their entries say nothing any more
        table = bt.clone()
        for b in range(B):
            for pg in range(width):
                if pg * PAGE >= sinks and (pg + 1) * PAGE <= done[b] + 1 - window:
                    table[b, pg] = 1 << 30
        md = attention.AbkvMetadataBuilder().build(0, SimpleNamespace(
            num_reqs=B, num_actual_tokens=T, query_start_loc=starts.to(DEV), query_start_loc_cpu=starts, seq_lens=now.to(DEV),
            _seq_lens_cpu=now, block_table_tensor=table.to(DEV), slot_mapping=sm.to(DEV), max_query_len=max(qlens),
            causal=True))
        out = torch.full((T, HKV * G * D), float("nan"), dtype=torch.bfloat16, device=DEV)
        impl.forward(None, q.to(DEV).view(T, -1), k.to(DEV).view(T, -1), v.to(DEV).view(T, -1), kv, md, out)
        at = 0
        for b, n in enumerate(qlens):
            seqs[b].append(k[at:at + n], v[at:at + n])
            o, A = seqs[b].attend(q[at:at + n], list(range(done[b], done[b] + n)), window, sinks)
            ref.check_out(out[at:at + n].view(n, HKV * G, D), o, A, (qlens, b))
            done[b] += n
            at += n

    for qlens in ([70, 33], [65, 1], [1, 90]) + ([1, 1],) * 8 + ([3, 2],):
        step(list(qlens))
    assert impl.workspace.read_error() == 0


def test_decode_and_eviction_on_two_streams():
    """Two sequences of calls at once on two streams, each with the workspace that its stream gets by itself."""
    g = torch.Generator().manual_seed(3)
    n, budget = 700, 300
    jobs = []
    for i in range(2):
        c = ref.Paged([n, n - 37], HKV, D, PAGE, 0, seed=20 + i)
        jobs.append(dict(c=c, kv=c.kv.to(DEV), bt=c.table.to(DEV), seq=c.seq.to(DEV), q=bf16(2, HKV * G, D, g=g).to(DEV)))

    def run(j):
        acc = torch.zeros((2, HKV, j["bt"].shape[1] * PAGE), device=DEV)
        kv, seq, outs = j["kv"].clone(), j["seq"], []
        for i in range(6):
            outs += decode.paged_decode_weighted([j["q"]], [kv], [j["bt"]], [seq], [acc])
            e = compaction.evict_by_weight([kv], [j["bt"]], [seq], [acc], budget=budget - 20 * i, num_recent=8)
            seq, acc = e.seq_lens[0], e.weights[0]
        return outs + [acc, seq]

    alone = [[t.clone() for t in run(j)] for j in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    for _ in range(3):
        got = []
        for j, s in zip(jobs, streams):
            with torch.cuda.stream(s):
                got.append(run(j))
        torch.cuda.synchronize()
        for a, b in zip(alone, got):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_a_cache_past_32_bit_offsets():
    """Pages behind 2^31 and 2^32 elements of the cache are read, written and moved where they lie."""
    g = torch.Generator().manual_seed(5)
    hkv, page = 8, 16
    per_page = 2 * page * hkv * D
    nb = (1 << 32) // per_page + 64
    kv = torch.empty((nb, 2, page, hkv, D), dtype=torch.bfloat16, device=DEV)
    n, width = 200, 13
    high = torch.randperm(40, generator=g)[:2 * width] + nb - 45
    bt = torch.stack([high[:width], high[width:]]).int()
    assert int(bt.min()) * per_page > (1 << 31)
    k, v = bf16(2, n, hkv, D, g=g), bf16(2, n, hkv, D, g=g)
    q = bf16(2, hkv, D, g=g)
    pos = torch.arange(n)
    sm = torch.cat([bt[b, pos // page].long() * page + pos % page for b in range(2)])
    btd, seq = bt.to(DEV), torch.tensor([n, n - 3], dtype=torch.int32, device=DEV)
    attention.store_kv(k.view(-1, hkv, D).to(DEV), v.view(-1, hkv, D).to(DEV), kv, sm.to(DEV))
    acc = torch.zeros((2, 1, width * page), device=DEV)
    qd = q.to(DEV)
    starts = torch.tensor([0, 1, 2], dtype=torch.int32, device=DEV)
    o1, = decode.paged_decode_weighted([qd], [kv], [btd], [seq], [acc], scale=SCALE)
    o2, lse = codestep.paged_prefill_window(qd, kv, btd, seq, starts, max_query_len=1, num_kv_heads=hkv, window=None,
                                            return_lse=True)
    w2 = torch.zeros_like(acc)
    codestep.paged_prompt_weights(qd, lse, kv, btd, seq, starts, w2, max_query_len=1, num_kv_heads=hkv)
    e = compaction.evict_by_weight([kv], [btd], [seq], [acc], budget=90, num_sinks=2, num_recent=5, return_keep=True)
    for b in range(2):
        m = n - 3 * b
        want = torch.zeros(m).double()
        for h in range(hkv):
            o, A, _, p = ref.attend(q[b:b + 1, h:h + 1], k[b, :m, h], v[b, :m, h], torch.ones(1, m, dtype=torch.bool), SCALE)
            ref.check_out(o1[b:b + 1, h:h + 1], o, A, ("decode", b, h))
            ref.check_out(o2[b:b + 1, h:h + 1], o, A, ("prompt", b, h))
            want += p[0, 0]
        for w in (acc, w2):
            assert (w[b, 0, :m].double().cpu() - want).abs().le(2.0 ** -11 * want).all()
        rows = e.keep[0][b, 0].cpu()
        assert (rows.numpy() == ref.evict_rows(acc[b, 0].cpu().numpy(), m, 90, 2, 5)).all()
        p90 = torch.arange(90)
        pg, off = bt[b, p90 // page].long().to(DEV), (p90 % page).to(DEV)
        assert torch.equal(kv[pg, 0, off].cpu(), k[b, rows.long()]) and torch.equal(kv[pg, 1, off].cpu(), v[b, rows.long()])


@pytest.mark.parametrize("layout", [0, 1])
def test_a_cache_of_two_blocks(layout):
    """Its shape fits both layouts: kv_layout says which."""
    c = ref.Paged([13], HKV, D, PAGE, layout, seed=9)
    kv, bt, seq = c.kv.to(DEV), c.table.to(DEV), c.seq.to(DEV)
    assert kv.shape[:2] == (2, 2)
    q = bf16(13, HKV * G, D, g=torch.Generator().manual_seed(9))
    starts = torch.tensor([0, 13], dtype=torch.int32, device=DEV)
    args = (kv, bt, seq, starts)
    kw = dict(max_query_len=13, num_kv_heads=HKV, window=5, num_sinks=1)
    with pytest.raises(ValueError, match="kv_layout"):
        codestep.paged_prefill_window(q.to(DEV), *args, **kw)
    out, lse = codestep.paged_prefill_window(q.to(DEV), *args, **kw, return_lse=True, kv_layout=layout)
    w = torch.zeros((1, HKV, PAGE), device=DEV)
    codestep.paged_prompt_weights(q.to(DEV), lse, *args, w, **kw, kv_layout=layout)
    with pytest.raises(ValueError, match="kv_layout"):
        compaction.evict_by_weight([kv], [bt], [seq], [w], budget=6)
    e = compaction.evict_by_weight([kv], [bt], [seq], [w], budget=6, return_keep=True, kv_layout=layout)
    s = Rows()
    s.append(c.K[0], c.V[0])
    o, A = s.attend(q, list(range(13)), 5, 1, count=13)
    ref.check_out(out, o, A)
    check_acc(w, [s], layout)
    K, V = c.rows(kv.cpu(), c.table, 0, 6)
    for h in range(HKV):
        rows = e.keep[0][0, h].cpu().long()
        assert (rows.numpy() == ref.evict_rows(w[0, h].cpu().numpy(), 13, 6, 0, 0)).all()
        assert torch.equal(K[:, h], c.K[0][rows, h]) and torch.equal(V[:, h], c.V[0][rows, h])
