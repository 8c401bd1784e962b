"""compaction.evict_by_weight on the GPU against a restatement in numpy (exact: rows are copied)."""
import numpy as np
import pytest
import torch

import bounded_ref as R
from abridgekv_b200 import _lib, compaction
from abridgekv_b200.workspace import Workspace

pytestmark = pytest.mark.gpu


def bits(t):
    return t.contiguous().view(torch.int16)


def make_weights(kind, shape, g):
    w = torch.rand(shape, generator=g)
    if kind == "ties":
        w = (w * 4).floor()
    elif kind == "heavy":
        w = torch.exp(-20 * w)
    elif kind == "wild":
        sel = torch.randint(0, 6, shape, generator=g)
        for i, v in enumerate((float("nan"), float("inf"), -float("inf"), 0.0, -0.0)):
            w = torch.where(sel == i, torch.full_like(w, v), w)
    elif kind == "signed":
        w = torch.randn(shape, generator=g) * 1e-3
    return w


def run(lens, Hkv, D, page, units, budget, sinks, recent, kind="rand", layout=0, dst=False, L=1, in_place_w=False, seed=0,
        workspace=None):
    g = torch.Generator().manual_seed(seed + 50)
    budgets = budget if isinstance(budget, list) else [budget] * L
    need = [sum((min(n, m) + page - 1) // page for n in lens) for m in budgets]
    caches = [R.Paged(lens, Hkv, D, page, layout, seed=seed + l, extra_pages=1 + (need[l] if dst else 0)) for l in range(L)]
    cap = max(1, max(lens)) + 3
    ws = [make_weights(kind, (len(lens), units, cap), g) for _ in range(L)]
    dst_tables = None
    if dst:
        dst_tables = []
        for l, c in enumerate(caches):
            used = set(c.table.flatten().tolist()) | {0}
            free = [p for p in range(c.nb) if p not in used]
            t = torch.zeros((len(lens), max(1, (min(max(lens), budgets[l]) + page - 1) // page)), dtype=torch.int32)
            for b, n in enumerate(lens):
                k = (min(n, budgets[l]) + page - 1) // page
                t[b, :k] = torch.tensor([free.pop() for _ in range(k)], dtype=torch.int32)
            dst_tables.append(t)
    kv = [c.kv.cuda() for c in caches]
    w_in = [w.cuda() for w in ws]
    res = compaction.evict_by_weight(kv, [c.table.cuda() for c in caches], [c.seq.cuda() for c in caches], w_in,
                                     budget=budget, num_sinks=sinks, num_recent=recent,
                                     dst_block_tables=[t.cuda() for t in dst_tables] if dst else None,
                                     return_keep=True, in_place_weights=in_place_w, workspace=workspace)
    for l, c in enumerate(caches):
        want = c.kv.clone()
        view = want if layout == 0 else want.transpose(0, 1)
        old = c.kv.clone() if layout == 0 else c.kv.transpose(0, 1).clone()
        W = torch.zeros_like(ws[l])
        K = np.full((len(lens), units, budgets[l]), -1)
        to = dst_tables[l] if dst else c.table
        for b, n in enumerate(lens):
            for u in range(units):
                keep = R.evict_rows(ws[l][b, u].numpy(), n, budgets[l], sinks, recent)
                K[b, u, :len(keep)] = keep
                W[b, u, :len(keep)] = ws[l][b, u, torch.from_numpy(keep)]
                hs = slice(None) if units == 1 else slice(u, u + 1)
                for i, r in enumerate(keep.tolist()):
                    view[to[b, i // page].long(), :, i % page, hs] = old[c.table[b, r // page].long(), :, r % page, hs]
        assert np.array_equal(res.keep[l].cpu().numpy(), K)
        assert torch.equal(res.seq_lens[l].cpu(), torch.tensor([min(n, budgets[l]) for n in lens], dtype=torch.int32))
        assert torch.equal(res.weights[l].cpu().view(torch.int32), W.view(torch.int32))
        assert torch.equal(bits(kv[l].cpu()), bits(want))
        if in_place_w:
            assert res.weights[l] is w_in[l]
        else:
            assert torch.equal(w_in[l].cpu().view(torch.int32), ws[l].view(torch.int32))
    return res


@pytest.mark.parametrize("dst", [False, True])
@pytest.mark.parametrize("kind", ["rand", "ties", "heavy", "wild", "signed"])
@pytest.mark.parametrize("Hkv,D,page,units", [(8, 128, 16, 1), (8, 128, 16, 8), (2, 64, 32, 2), (1, 64, 16, 1)])
def test_select_and_move(dst, kind, Hkv, D, page, units):
    run([0, 1, 40, 64, 65, 300, 257], Hkv, D, page, units, 64, 4, 16, kind=kind, dst=dst)


@pytest.mark.parametrize("dst", [False, True])
@pytest.mark.parametrize("budget,sinks,recent", [(1, 0, 0), (1, 1, 0), (1, 0, 1), (20, 10, 10), (33, 0, 0), (99, 0, 50),
                                                 (100, 4, 4), (500, 3, 3)])
def test_budgets(dst, budget, sinks, recent):
    run([100, 101, 30], 4, 64, 16, 4, budget, sinks, recent, dst=dst)


@pytest.mark.parametrize("dst", [False, True])
@pytest.mark.parametrize("Hkv", [1, 2, 4, 8])
@pytest.mark.parametrize("D", [64, 128])
def test_heads_and_layouts(dst, Hkv, D):
    run([130, 77], Hkv, D, 16, Hkv, 50, 2, 8, dst=dst, layout=1)
    run([130, 77], Hkv, D, 64, 1, 50, 2, 8, dst=dst, layout=1, in_place_w=True)


def test_layers_with_their_own_budgets():
    run([200, 90], 2, 64, 16, 2, [128, 64, 100], 4, 8, L=3)
    run([200, 90], 2, 64, 16, 1, [128, 64, 100], 4, 8, L=3, dst=True, in_place_w=True)
    run([33], 1, 64, 16, 1, 20, 1, 1, L=50)


@pytest.mark.parametrize("n,budget", [(5000, 4999), (5000, 2500), (9000, 8300)])
def test_in_place_across_many_chunks(n, budget):
    run([n, 700], 2, 64, 16, 2, budget, 4, 64, in_place_w=True)


def test_longer_than_the_key_cache():
    """Past the keys that fit shared memory the weights are read again for every pass."""
    n = 52000
    g = torch.Generator().manual_seed(1)
    page, nb = 64, (n + 63) // 64 + 1
    kv = torch.randn((nb, 2, page, 1, 64), generator=g).to(torch.bfloat16)
    table = (torch.randperm(nb - 1, generator=g) + 1).int()[None]
    w = make_weights("ties", (1, 1, n), g) + make_weights("heavy", (1, 1, n), g)
    res = compaction.evict_by_weight([kv.cuda()], [table.cuda()], [torch.tensor([n], dtype=torch.int32).cuda()], [w.cuda()],
                                     budget=30000, num_sinks=4, num_recent=100, return_keep=True)
    keep = R.evict_rows(w[0, 0].numpy(), n, 30000, 4, 100)
    assert np.array_equal(res.keep[0][0, 0].cpu().numpy(), keep)


def test_reports_bad_lengths_and_pages():
    c = R.Paged([40], 1, 64, 16, seed=3)
    w = torch.rand((1, 1, 30))
    ws = Workspace("cuda:0")
    res = compaction.evict_by_weight([c.kv.cuda()], [c.table.cuda()], [c.seq.cuda()], [w.cuda()], budget=20, workspace=ws)
    assert ws.read_error() == 2 and int(res.seq_lens[0]) == 20  # 40 rows, 30 weights
    bad = c.table.clone()
    bad[0, 1] = 99
    kv = c.kv.cuda()
    compaction.evict_by_weight([kv], [bad.cuda()], [c.seq.cuda()], [torch.rand((1, 1, 48)).cuda()], budget=20, workspace=ws)
    assert ws.read_error() == 1
    neg = torch.tensor([-5], dtype=torch.int32).cuda()
    res = compaction.evict_by_weight([kv], [c.table.cuda()], [neg], [torch.rand((1, 1, 48)).cuda()], budget=20, workspace=ws)
    assert ws.read_error() == 2 and int(res.seq_lens[0]) == 0


def test_graph_replay():
    c = R.Paged([300, 150], 4, 128, 16, seed=5)
    w0 = torch.rand((2, 4, 304)).cuda()
    kv0 = c.kv.cuda()
    table, seq = c.table.cuda(), c.seq.cuda()
    kv, w = kv0.clone(), w0.clone()
    ref = compaction.evict_by_weight([kv], [table], [seq], [w], budget=100, num_sinks=4, num_recent=20, in_place_weights=True)
    kv2, w2 = kv0.clone(), w0.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = compaction.evict_by_weight([kv2], [table], [seq], [w2], budget=100, num_sinks=4, num_recent=20,
                                         in_place_weights=True)
    for _ in range(2):
        kv2.copy_(kv0), w2.copy_(w0)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(bits(kv2), bits(kv)) and torch.equal(w2, w) and torch.equal(got.seq_lens[0], ref.seq_lens[0])


def test_refusals():
    c = R.Paged([40], 2, 64, 16, seed=7)
    kv, bt, sl, w = [c.kv.cuda()], [c.table.cuda()], [c.seq.cuda()], [torch.rand((1, 2, 48)).cuda()]
    ev = compaction.evict_by_weight
    for kw in (dict(budget=0), dict(budget=8, num_sinks=5, num_recent=4), dict(budget=8, num_sinks=-1),
               dict(budget=[8, 9])):
        with pytest.raises(ValueError, match="budget"):
            ev(kv, bt, sl, w, **kw)
    with pytest.raises(TypeError, match="weights"):
        ev(kv, bt, sl, [w[0].double()], budget=8)
    with pytest.raises(ValueError, match="weights"):
        ev(kv, bt, sl, [w[0][:, :, ::2]], budget=8)
    with pytest.raises(ValueError, match="row per KV head"):
        ev(kv, bt, sl, [torch.rand((1, 3, 48)).cuda()], budget=8)
    with pytest.raises(ValueError, match="its own cache"):
        ev(kv * 2, bt * 2, sl * 2, w * 2, budget=8)
    with pytest.raises(TypeError, match="2-byte"):
        ev([kv[0].float()], bt, sl, w, budget=8)
    with pytest.raises(TypeError, match="block_table"):
        ev(kv, [bt[0].long()], sl, w, budget=8)
    with pytest.raises(_lib.AbkvError):
        ev(kv, bt, sl, w, budget=8, dst_block_tables=bt)
    with pytest.raises(_lib.AbkvError):
        ev([torch.zeros((4, 2, 16, 2, 32), dtype=torch.bfloat16, device="cuda")], bt, sl, w, budget=8)


def test_a_budget_far_above_the_rows_needs_no_memory_for_it():
    c = R.Paged([40, 7], 2, 64, 16, 0, seed=4)
    kv, bt, seq = c.kv.cuda(), c.table.cuda(), c.seq.cuda()
    before, w = kv.clone(), torch.rand((2, 2, 48), device="cuda")
    ws = Workspace("cuda", 4096)
    e = compaction.evict_by_weight([kv], [bt], [seq], [w], budget=1 << 30, num_sinks=4, num_recent=100, workspace=ws)
    assert ws.nbytes < 1 << 20 and e.seq_lens[0].tolist() == [40, 7]
    assert torch.equal(kv.nan_to_num(7.0), before.nan_to_num(7.0))
    for b, n in enumerate((40, 7)):
        assert torch.equal(e.weights[0][b, :, :n], w[b, :, :n]) and (e.weights[0][b, :, n:] == 0).all()


def test_a_destination_without_room_is_refused():
    c = R.Paged([40], 2, 64, 16, seed=7)
    kv, bt, sl, w = [c.kv.cuda()], [c.table.cuda()], [c.seq.cuda()], [torch.rand((1, 2, 48)).cuda()]
    before = bits(kv[0]).clone()
    for width, budget in ((1, 17), (2, 33), (2, 1000)):
        with pytest.raises(ValueError, match="dst_block_table"):
            compaction.evict_by_weight(kv, bt, sl, w, budget=budget, dst_block_tables=[bt[0][:, :width].contiguous()])
    assert torch.equal(bits(kv[0]), before)
