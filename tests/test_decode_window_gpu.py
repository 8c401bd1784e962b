"""paged_decode_window / paged_decode_weighted on the GPU against a 64-bit restatement."""
import pytest
import torch

import bounded_ref as R
from abridgekv_b200 import decode
from abridgekv_b200.workspace import Workspace

pytestmark = pytest.mark.gpu


def cuda(ts):
    return [t.cuda() for t in ts]


def oracle(cache, q, b, window, sinks, scale):
    """out, A [Hq, D] and p [Hkv, G, n] of sequence b."""
    n, Hkv = cache.lens[b], cache.Hkv
    G = q.shape[1] // Hkv
    if n == 0:
        z = torch.zeros((q.shape[1], q.shape[2]), dtype=torch.float64)
        return z, z, torch.zeros((Hkv, G, 0), dtype=torch.float64)
    vis = R.visible([n - 1], n, window, sinks)
    o, a, p = [], [], []
    for h in range(Hkv):
        oh, ah, _, ph = R.attend(q[b:b + 1, h * G:(h + 1) * G], cache.K[b][:, h], cache.V[b][:, h], vis, scale)
        o.append(oh[0]), a.append(ah[0]), p.append(ph[0])
    return torch.cat(o), torch.cat(a), torch.stack(p)


def run(lens, Hkv, G, D, page, window, sinks, L=1, chunk=0, weights=None, seed=0, workspace=None):
    caches = [R.Paged(lens, Hkv, D, page, seed=seed + l) for l in range(L)]
    g = torch.Generator().manual_seed(seed + 100)
    qs = [torch.randn((len(lens), Hkv * G, D), generator=g).to(torch.bfloat16) for _ in range(L)]
    win = window if isinstance(window, (list, tuple)) else [window] * L
    snk = sinks if isinstance(sinks, (list, tuple)) else [sinks] * L
    scale = D ** -0.5
    args = (cuda(qs), cuda([c.kv for c in caches]), cuda([c.table for c in caches]), cuda([c.seq for c in caches]))
    kw = dict(window=window, num_sinks=sinks, chunk_tokens=chunk, workspace=workspace)
    if weights is None:
        outs = decode.paged_decode_window(*args, **kw)
        w0 = w1 = None
    else:
        units = Hkv if weights == "head" else 1
        cap = max(1, max(lens)) + 5
        w0 = [torch.rand((len(lens), units, cap), generator=g) for _ in range(L)]
        w1 = cuda(w0)
        outs = decode.paged_decode_weighted(*args, w1, **kw)
    for l in range(L):
        for b, n in enumerate(lens):
            o, a, p = oracle(caches[l], qs[l], b, win[l] or 0, snk[l], scale)
            R.check_out(outs[l][b], o, a, (l, b, n))
            if w0 is not None:
                add = torch.zeros(w0[l].shape[1:], dtype=torch.float64)
                add[:, :n] = p.sum(1) if weights == "head" else p.sum((0, 1))[None]
                R.check_weights(w1[l][b], w0[l][b], add, (l, b, n))
                assert torch.equal(w1[l][b, :, n:].cpu(), w0[l][b, :, n:])
    return outs, w1


LENS = [1, 0, 16, 17, 100, 333]


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (33, 4), (40, 70), (64, 16), (100, 1), (400, 4),
                                          (None, 9)])
@pytest.mark.parametrize("Hkv,G,D,page", [(8, 4, 128, 16), (2, 3, 64, 32)])
def test_window(window, sinks, Hkv, G, D, page):
    run(LENS, Hkv, G, D, page, window, sinks)


@pytest.mark.parametrize("Hkv", [1, 2, 4, 8])
@pytest.mark.parametrize("G", [1, 8])
@pytest.mark.parametrize("weights", ["head", "all"])
@pytest.mark.parametrize("window,sinks", [(None, 0), (37, 5)])
def test_weights_heads(Hkv, G, weights, window, sinks):
    run([200, 7, 0, 65], Hkv, G, 128, 16, window, sinks, weights=weights)


@pytest.mark.parametrize("chunk", [16, 48, 128, 0])
def test_chunks_and_layers(chunk):
    """Every split of the rows, layers with their own windows, more layers than one launch of scores."""
    run([500, 31, 260], 4, 2, 64, 16, [None, 50, 128], [0, 3, 20], L=3, chunk=chunk, weights="head")
    run([500, 31, 260], 8, 2, 128, 64, [None, 50, 128], [0, 3, 20], L=3, chunk=chunk, weights="all")


def test_many_layers_one_launch_or_more():
    run([40, 3], 2, 2, 64, 16, 20, 2, L=60)
    run([40, 3], 2, 2, 64, 16, 20, 2, L=60, weights="head")


def test_unlimited_window_equals_paged_decode():
    lens = [300, 16, 77]
    c = R.Paged(lens, 8, 128, 16, seed=3)
    q = torch.randn((3, 32, 128), generator=torch.Generator().manual_seed(4)).to(torch.bfloat16).cuda()
    args = ([q], [c.kv.cuda()], [c.table.cuda()], [c.seq.cuda()])
    a = decode.paged_decode(*args, chunk_tokens=64)[0]
    b = decode.paged_decode_window(*args, window=None, chunk_tokens=64)[0]
    assert torch.equal(a, b)


def test_freed_pages_are_not_read():
    """Pages without a visible row may hold any id and any content."""
    lens, page, window, sinks = [400, 123], 16, 50, 3
    c = R.Paged(lens, 4, 128, page, seed=5)
    q = torch.randn((2, 16, 128), generator=torch.Generator().manual_seed(6)).to(torch.bfloat16)
    kv, table = c.kv.cuda(), c.table.clone()
    ref = decode.paged_decode_window([q.cuda()], [kv], [table.cuda()], [c.seq.cuda()], window=window, num_sinks=sinks)
    for b, n in enumerate(lens):
        dead = [t for t in range((n + page - 1) // page) if t * page >= sinks and (t + 1) * page <= n - window]
        assert dead
        for t in dead:
            table[b, t] = -7
    ws = Workspace("cuda:0")
    got = decode.paged_decode_window([q.cuda()], [kv], [table.cuda()], [c.seq.cuda()], window=window, num_sinks=sinks,
                                     workspace=ws)
    assert torch.equal(ref[0], got[0]) and ws.read_error() == 0


def test_repeat_is_bitwise_and_accumulates():
    c = R.Paged([700, 90], 4, 128, 16, seed=8)
    q = torch.randn((2, 16, 128), generator=torch.Generator().manual_seed(9)).to(torch.bfloat16).cuda()
    args = ([q], [c.kv.cuda()], [c.table.cuda()], [c.seq.cuda()])
    once = [torch.zeros((2, 4, 704), device="cuda")]
    decode.paged_decode_weighted(*args, once)
    again = [torch.zeros((2, 4, 704), device="cuda")]
    decode.paged_decode_weighted(*args, again)
    assert torch.equal(once[0], again[0])
    decode.paged_decode_weighted(*args, again)
    assert torch.equal(again[0], 2 * once[0])
    for b, n in enumerate(c.lens):  # every head's weights of a sequence sum to one
        assert torch.allclose(once[0][b, :, :n].sum(-1), torch.full((4,), 4.0, device="cuda"), rtol=1e-5, atol=0)


def test_strided_weights_of_a_larger_pool():
    lens = [50, 130]
    c = R.Paged(lens, 2, 64, 16, seed=11)
    q = torch.randn((2, 4, 64), generator=torch.Generator().manual_seed(12)).to(torch.bfloat16).cuda()
    pool = torch.zeros((3, 2, 2, 160), device="cuda")  # [units+1][B][2][rows]: units outermost
    w = pool[:2, :, 0].transpose(0, 1)
    dense = torch.zeros((2, 2, 160), device="cuda")
    args = ([q], [c.kv.cuda()], [c.table.cuda()], [c.seq.cuda()])
    decode.paged_decode_weighted(*args, [w])
    decode.paged_decode_weighted(*args, [dense])
    assert torch.equal(w, dense)
    assert not pool[2].any() and not pool[:, :, 1].any()


def test_short_weights_are_cut_and_reported():
    c = R.Paged([60], 2, 64, 16, seed=13)
    q = torch.randn((1, 4, 64), generator=torch.Generator().manual_seed(14)).to(torch.bfloat16).cuda()
    w = torch.zeros((1, 2, 64), device="cuda")
    ws = Workspace("cuda:0")
    decode.paged_decode_weighted([q], [c.kv.cuda()], [c.table.cuda()], [c.seq.cuda()], [w[:, :, :40]], workspace=ws)
    assert ws.read_error() == 2 and not w[:, :, 40:].any()
    sums = w[:, :, :40].sum(-1)
    assert torch.allclose(sums, torch.full_like(sums, 2.0), rtol=1e-5, atol=0)


def test_graph_replay_and_side_stream():
    c = R.Paged([300, 45], 8, 128, 16, seed=15)
    q = torch.randn((2, 32, 128), generator=torch.Generator().manual_seed(16)).to(torch.bfloat16).cuda()
    args = ([q], [c.kv.cuda()], [c.table.cuda()], [c.seq.cuda()])
    w = torch.zeros((2, 8, 304), device="cuda")
    ref = decode.paged_decode_weighted(*args, [w], window=64, num_sinks=4)[0].clone()
    wref = w.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    w2 = torch.zeros_like(w)
    side.wait_stream(torch.cuda.current_stream())
    got = decode.paged_decode_weighted(*args, [w2], window=64, num_sinks=4, stream=side)[0]
    torch.cuda.synchronize()
    assert torch.equal(got, ref) and torch.equal(w2, wref)
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        o1 = decode.paged_decode_weighted(*args, [w], window=64, num_sinks=4)[0]
    with torch.cuda.graph(g2):
        o2 = decode.paged_decode_window(*args, window=100, num_sinks=1)[0]
    ref2 = decode.paged_decode_window(*args, window=100, num_sinks=1)[0]
    for _ in range(3):
        w.zero_(), o1.zero_(), o2.zero_()
        g1.replay(), g2.replay()
        torch.cuda.synchronize()
        assert torch.equal(o1, ref) and torch.equal(w, wref) and torch.equal(o2, ref2)


def test_refusals():
    c = R.Paged([60], 2, 64, 16, seed=17)
    q = torch.zeros((1, 4, 64), dtype=torch.bfloat16, device="cuda")
    args = ([q], [c.kv.cuda()], [c.table.cuda()], [c.seq.cuda()])
    w = torch.zeros((1, 2, 64), device="cuda")
    with pytest.raises(ValueError, match="window"):
        decode.paged_decode_window(*args, window=-1)
    with pytest.raises(ValueError, match="per layer"):
        decode.paged_decode_window(*args, window=[3, 4])
    with pytest.raises(ValueError, match="num_sinks"):
        decode.paged_decode_window(*args, window=3, num_sinks=-2)
    with pytest.raises(TypeError, match="weights"):
        decode.paged_decode_weighted(*args, [w.half()])
    with pytest.raises(ValueError, match="weights"):
        decode.paged_decode_weighted(*args, [w.expand(1, 2, 64)[:, :, ::2]])
    with pytest.raises(ValueError, match="row per KV head"):
        decode.paged_decode_weighted(*args, [torch.zeros((1, 3, 64), device="cuda")])
    with pytest.raises(ValueError, match="overlap"):
        decode.paged_decode_weighted(*args, [torch.zeros((1, 1, 64), device="cuda").expand(1, 2, 64)])
    with pytest.raises(RuntimeError, match="unsupported|UNSUPPORTED|invalid"):
        decode.paged_decode_window(*args, window=3, chunk_tokens=24)
