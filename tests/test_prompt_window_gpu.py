"""paged_prefill_window and paged_prompt_weights on the GPU against a 64-bit restatement."""
import pytest
import torch

import bounded_ref as R
from abridgekv_b200 import codestep
from abridgekv_b200.workspace import Workspace

pytestmark = pytest.mark.gpu
D = 128


class Case:
    def __init__(self, qlens, lens, Hkv, G, page=16, layout=0, seed=0, pad_rows=0):
        self.c = R.Paged(lens, Hkv, D, page, layout, seed=seed)
        self.qlens, self.Hkv, self.G = qlens, Hkv, G
        self.T = sum(qlens) + pad_rows
        g = torch.Generator().manual_seed(seed + 100)
        self.q = torch.randn((self.T, Hkv * G, D), generator=g).to(torch.bfloat16)
        qs = [0]
        for x in qlens:
            qs.append(qs[-1] + x)
        self.qs = qs
        self.args = (self.q.cuda(), self.c.kv.cuda(), self.c.table.cuda(), self.c.seq.cuda(),
                     torch.tensor(qs, dtype=torch.int32).cuda())

    def oracle(self, window, sinks, scale=D ** -0.5):
        """Per request: out, A, lse [nq, Hq, ..], p [Hkv][nq, G, n]."""
        res = []
        for r, (nq, n) in enumerate(zip(self.qlens, self.c.lens)):
            vis = R.visible(list(range(n - nq, n)), n, window, sinks)
            q = self.q[self.qs[r]:self.qs[r + 1]]
            parts = [R.attend(q[:, h * self.G:(h + 1) * self.G], self.c.K[r][:, h], self.c.V[r][:, h], vis, scale)
                     for h in range(self.Hkv)]
            res.append(([torch.cat([x[i] for x in parts], 1) for i in range(3)], [x[3] for x in parts]))
        return res


def run(qlens, lens, Hkv, G, window, sinks, page=16, layout=0, observe=None, units=None, seed=0, pad_rows=0):
    case = Case(qlens, lens, Hkv, G, page, layout, seed, pad_rows)
    ws = Workspace("cuda:0")
    kw = dict(max_query_len=max(qlens), num_kv_heads=Hkv, window=window, num_sinks=sinks, workspace=ws)
    out = torch.full((case.T, Hkv * G, D), 7.0, dtype=torch.bfloat16, device="cuda")
    got, lse = codestep.paged_prefill_window(*case.args, out=out, return_lse=True, **kw)
    ref = case.oracle(window or 0, sinks)
    for r in range(len(qlens)):
        (o, a, l), _ = ref[r]
        sl = slice(case.qs[r], case.qs[r + 1])
        R.check_out(got[sl], o, a, (r, qlens[r], case.c.lens[r]))
        # log-sum-exp: 32-bit scores (2^-13 of relative weight) and a 32-bit sum
        assert ((lse[sl].double().cpu() - l).abs() <= 2.0 ** -12 + 2.0 ** -22 * l.abs()).all(), r
    assert (got[case.qs[-1]:] == 7.0).all()
    cap = max(case.c.lens) + 4
    for u in ([units] if units else sorted({1, Hkv})):
        w0 = torch.rand((len(qlens), u, cap), generator=torch.Generator().manual_seed(seed))
        w = w0.cuda()
        codestep.paged_prompt_weights(case.args[0], lse, *case.args[1:], w, observe=observe, **kw)
        for r, (nq, n) in enumerate(zip(qlens, case.c.lens)):
            add = torch.zeros((u, cap), dtype=torch.float64)
            for h, p in enumerate(ref[r][1]):
                part = p[nq - min(nq, observe or nq):].sum((0, 1))
                add[h if u > 1 or Hkv == 1 else 0, :n] += part
            # lse rounded to 32 bits enters each weight once more
            R.check_weights(w[r], w0[r], add, (r, u))
            assert torch.equal(w[r, :, n:].cpu(), w0[r, :, n:])
    assert ws.read_error() == 0


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 3), (64, 0), (100, 4), (130, 70), (128, 64), (17, 200), (500, 1),
                                          (None, 5)])
@pytest.mark.parametrize("layout", [0, 1])
def test_window(window, sinks, layout):
    run([1, 130, 64, 300], [1, 130, 200, 700], 2, 2, window, sinks, layout=layout, pad_rows=5)


@pytest.mark.parametrize("Hkv", [1, 2, 4, 8])
@pytest.mark.parametrize("G", [1, 3, 4, 8])
def test_heads(Hkv, G):
    run([40, 1], [300, 77], Hkv, G, 90, 10, page=32)
    run([40, 9], [40, 300], Hkv, G, None, 0, page=64, observe=7)


@pytest.mark.parametrize("window,sinks", [(None, 0), (60, 4), (200, 65), (31, 0)])
@pytest.mark.parametrize("observe", [1, 5, 32, 33, 100, None])
def test_observe(window, sinks, observe):
    run([150, 3, 64], [420, 500, 64], 2, 4, window, sinks, observe=observe)


@pytest.mark.parametrize("shift", range(0, 64, 7))
def test_boundaries_inside_tiles(shift):
    """Window starts, sink ends and lengths at every kind of offset inside a 64-row tile."""
    run([129, 20], [400 + shift, 333 - shift], 1, 2, 70 + shift, shift, seed=shift)


def test_many_items():
    """More work items than CTAs, ragged lengths."""
    run([700, 33, 257], [1500, 33, 1300], 8, 2, None, 0)
    run([700, 33, 257], [1500, 33, 1300], 8, 2, 300, 20, units=8)


def test_freed_pages_are_not_read():
    window, sinks = 100, 20
    case = Case([30, 130], [500, 700], 4, 2, seed=3)
    ws = Workspace("cuda:0")
    kw = dict(max_query_len=130, num_kv_heads=4, window=window, num_sinks=sinks, workspace=ws)
    ref, lse = codestep.paged_prefill_window(*case.args, return_lse=True, **kw)
    w = torch.zeros((2, 4, 700), device="cuda")
    codestep.paged_prompt_weights(case.args[0], lse, *case.args[1:], w, **kw)
    table = case.c.table.clone()
    for r, (nq, n) in enumerate(zip(case.qlens, case.c.lens)):
        for t in range((n + 15) // 16):
            if t * 16 >= sinks and (t + 1) * 16 <= n - nq - window + 1:
                table[r, t] = 0 if t % 2 else -3  # the null block (NaN rows), or no page at all
    args = (case.args[0], case.args[1], table.cuda(), *case.args[3:])
    got, lse2 = codestep.paged_prefill_window(*args, return_lse=True, **kw)
    w2 = torch.zeros_like(w)
    codestep.paged_prompt_weights(args[0], lse, *args[1:], w2, **kw)
    assert torch.equal(ref, got) and torch.equal(lse, lse2) and torch.equal(w, w2) and ws.read_error() == 0


def test_no_window_equals_paged_prefill():
    case = Case([200, 65], [333, 65], 4, 2, seed=5)
    a = codestep.paged_prefill(*case.args, max_query_len=200, num_kv_heads=4)
    b = codestep.paged_prefill_window(*case.args, max_query_len=200, num_kv_heads=4, window=None)
    assert torch.equal(a, b)


def test_strided_query_and_repeat():
    case = Case([100, 30], [260, 90], 2, 4, seed=6)
    wide = torch.zeros((case.T, 2, 8, D), dtype=torch.bfloat16, device="cuda")
    wide[:, 1] = case.args[0]
    kw = dict(max_query_len=100, num_kv_heads=2, window=50, num_sinks=4)
    a, la = codestep.paged_prefill_window(*case.args, return_lse=True, **kw)
    b, lb = codestep.paged_prefill_window(wide[:, 1], *case.args[1:], return_lse=True, **kw)
    assert torch.equal(a, b) and torch.equal(la, lb)
    ws = [torch.zeros((2, u, 260), device="cuda") for u in (1, 1, 2, 2)]
    for i, q in enumerate((case.args[0], wide[:, 1]) * 2):
        codestep.paged_prompt_weights(q, la, *case.args[1:], ws[i], **kw)
    assert torch.equal(ws[0], ws[1]) and torch.equal(ws[2], ws[3])
    # the counted rows' weights sum to one per row and head
    tot = ws[2].sum(-1).cpu()
    assert torch.allclose(tot, torch.tensor([[400.0, 400.0], [120.0, 120.0]]), rtol=1e-5)


def test_bad_device_values_are_reported():
    case = Case([30], [90], 2, 2, seed=7)
    q, kv, bt, sl, qs = case.args
    ws = Workspace("cuda:0")
    kw = dict(max_query_len=30, num_kv_heads=2, window=40, num_sinks=4, workspace=ws)
    out, lse = codestep.paged_prefill_window(*case.args, return_lse=True, **kw)
    w = torch.zeros((1, 2, 90), device="cuda")
    codestep.paged_prompt_weights(q, lse, kv, bt, torch.full_like(sl, 20), qs, w, **kw)
    assert ws.read_error() == 2 and not w.any()  # fewer cache rows than query rows
    codestep.paged_prompt_weights(q, lse, kv, bt, sl, qs, w[:, :, :50], **kw)
    assert ws.read_error() == 2 and not w.any()
    codestep.paged_prompt_weights(q, lse, kv, bt, sl, torch.tensor([0, 31], dtype=torch.int32).cuda(), w, **kw)
    assert ws.read_error() == 16 and not w.any()
    codestep.paged_prompt_weights(q, lse, kv, bt, sl, qs, w, **{**kw, "max_query_len": 8})
    assert ws.read_error() == 16  # only the last 8 rows were counted
    assert torch.allclose(w.sum(-1).cpu(), torch.full((1, 2), 16.0), rtol=1e-5)
    bad = bt.clone()
    bad[0, 5] = 1000
    codestep.paged_prefill_window(q, kv, bad, sl, qs, **kw)
    assert ws.read_error() == 1
    codestep.paged_prompt_weights(q, lse, kv, bad, sl, qs, w, **kw)
    assert ws.read_error() == 1


def test_graphs():
    case = Case([100, 30], [260, 90], 4, 4, seed=8)
    kw = dict(max_query_len=100, num_kv_heads=4, window=50, num_sinks=4)
    ref, lref = codestep.paged_prefill_window(*case.args, return_lse=True, **kw)
    wref = codestep.paged_prompt_weights(case.args[0], lref, *case.args[1:], torch.zeros((2, 1, 260), device="cuda"), **kw)
    w = torch.zeros((2, 1, 260), device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out, lse = codestep.paged_prefill_window(*case.args, return_lse=True, **kw)
        codestep.paged_prompt_weights(case.args[0], lse, *case.args[1:], w, **kw)
    for _ in range(2):
        w.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ref) and torch.equal(lse, lref) and torch.equal(w, wref)


def test_refusals():
    case = Case([30], [90], 2, 2, seed=9)
    kw = dict(max_query_len=30, num_kv_heads=2)
    with pytest.raises(ValueError, match="window"):
        codestep.paged_prefill_window(*case.args, window=-1, **kw)
    with pytest.raises(ValueError, match="max_query_len"):
        codestep.paged_prefill_window(*case.args, window=4, max_query_len=0, num_kv_heads=2)
    with pytest.raises(TypeError, match="CUDA"):
        codestep.paged_prefill_window(case.q, *case.args[1:], window=4, **kw)
    lse, w = torch.zeros((30, 4), device="cuda"), torch.zeros((1, 2, 90), device="cuda")
    pw = codestep.paged_prompt_weights
    with pytest.raises(ValueError, match="observe"):
        pw(case.args[0], lse, *case.args[1:], w, observe=0, **kw)
    with pytest.raises(ValueError, match="lse"):
        pw(case.args[0], lse[:, :3], *case.args[1:], w, **kw)
    with pytest.raises(TypeError, match="weights"):
        pw(case.args[0], lse, *case.args[1:], w.double(), **kw)
    with pytest.raises(ValueError, match="weights"):
        pw(case.args[0], lse, *case.args[1:], torch.zeros((1, 3, 90), device="cuda"), **kw)
    with pytest.raises(ValueError, match="overlap"):
        pw(case.args[0], lse, *case.args[1:], torch.zeros((1, 1, 90), device="cuda").expand(1, 2, 90), **kw)


@pytest.mark.parametrize("observe", [None, 32])
def test_rows_of_a_bad_page_collect_nothing(observe):
    """Their scores come from whatever was loaded there before, and the accumulators outlive the call.  (Nor do the rows
    behind it in its tile of 128.)"""
    case = Case([300, 40], [700, 333], 2, 2, seed=12)
    q, kv, bt, sl, qs = case.args
    kw = dict(max_query_len=300, num_kv_heads=2, window=None, observe=observe)
    ws = Workspace("cuda:0")
    _, lse = codestep.paged_prefill_window(*case.args, max_query_len=300, num_kv_heads=2, window=None, return_lse=True)
    bad = bt.clone()
    holes = [(0, 2), (0, 30), (1, 0), (1, 20)]
    for r, slot in holes:
        bad[r, slot] = 10 ** 6
    for units in (2, 1):
        w0 = torch.rand((2, units, 720), generator=torch.Generator().manual_seed(1)).cuda()
        want, w = w0.clone(), w0.clone()
        codestep.paged_prompt_weights(q, lse, kv, bt, sl, qs, want, **kw)
        codestep.paged_prompt_weights(q, lse, kv, bad, sl, qs, w, workspace=ws, **kw)
        assert ws.read_error() == 1
        for r, slot in holes:
            s = slice(16 * slot, (16 * slot // 128 + 1) * 128)
            want[r, :, s] = w0[r, :, s]
        assert torch.equal(w, want)


def test_other_head_sizes_are_refused_before_the_launch():
    q = torch.zeros((4, 4, 64), dtype=torch.bfloat16, device="cuda")
    kv = torch.zeros((5, 2, 16, 2, 64), dtype=torch.bfloat16, device="cuda")
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    args, kw = (kv, i32(1).view(1, 1), i32(4), i32(0, 4)), dict(max_query_len=4, num_kv_heads=2, window=3)
    with pytest.raises(NotImplementedError, match="128"):
        codestep.paged_prefill_window(q, *args, **kw)
    with pytest.raises(NotImplementedError, match="128"):
        codestep.paged_prompt_weights(q, torch.zeros((4, 4), device="cuda"), *args, torch.zeros((1, 2, 16), device="cuda"), **kw)
