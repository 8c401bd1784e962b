"""prefill.window_attention (forward and backward) on the GPU against 64-bit formulas.

Bounds, elementwise (u = 2^-8, half a bf16 step; e = 2^-12 for everything in 32 bits, as in bounded_ref):
* out: bounded_ref.check_out.
* dV = P^T dO with P rounded to bf16: (u + e) sum P |dO| + u |dV|.
* dS = P (dP - Di), Di = sum dO O of the bf16 output (error u sum |dO| |O|), dS rounded to bf16:
  d = u (|dS| + P sum |dO| |O|) + e P (|dP| + |Di|); dQ and dK multiply it out: scale d |K| + u |dQ|, scale d^T |Q| + u |dK|.
"""
import pytest
import torch

import bounded_ref as R
from abridgekv_b200 import prefill
from abridgekv_b200.workspace import Workspace

pytestmark = pytest.mark.gpu
U, E = R.U16, R.U32


def formulas(q, k, v, do, window, sinks, scale):
    """64-bit out, dq, dk, dv and their bounds (A of out; the rest elementwise)."""
    q, k, v, do = (t.double() for t in (q, k, v, do))
    B, H, S, D = q.shape
    G = H // k.shape[1]
    K, V = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
    vis = R.visible(list(range(S)), S, window, sinks)
    x = (q @ K.transpose(2, 3) * scale).masked_fill(~vis, float("-inf"))
    P = torch.softmax(x, -1)
    O = P @ V
    dP = do @ V.transpose(2, 3)
    Di = (do * O).sum(-1, keepdim=True)
    dS = P * (dP - Di)
    d = U * (dS.abs() + P * (do.abs() * O.abs()).sum(-1, keepdim=True)) + E * P * (dP.abs() + Di.abs())

    def heads(t):
        return t.reshape(B, H // G, G, S, D).sum(2)

    dq, dk, dv = scale * dS @ K, heads(scale * dS.transpose(2, 3) @ q), heads(P.transpose(2, 3) @ do)
    return (O, P @ V.abs()), ((dq, scale * d @ K.abs() + U * dq.abs()),
                              (dk, heads(scale * d.transpose(2, 3) @ q.abs()) + U * dk.abs()),
                              (dv, heads((U + E) * P.transpose(2, 3) @ do.abs()) + U * dv.abs())), x.logsumexp(-1)


def inputs(B, H, Hkv, S, D, seed=0, bshd=True):
    g = torch.Generator().manual_seed(seed)
    mk = lambda h: (torch.randn((B, S, h, D), generator=g).to(torch.bfloat16).transpose(1, 2) if bshd else  # noqa: E731
                    torch.randn((B, h, S, D), generator=g).to(torch.bfloat16))
    return mk(H), mk(Hkv), mk(Hkv), mk(H)


def check(got, pairs, tag):
    for name, t, (ref, bound) in zip(("dq", "dk", "dv"), got, pairs):
        t = t.double().cpu()
        assert not torch.isnan(t).any(), (tag, name)
        worst = ((t - ref).abs() / (bound + 1e-30)).max()
        assert worst <= 1, (tag, name, float(worst))


def run(B, H, Hkv, S, D, window, sinks, scale=None, seed=0, bshd=True):
    q, k, v, do = inputs(B, H, Hkv, S, D, seed, bshd)
    (O, A), grads, lse = formulas(q, k, v, do, window, sinks, scale or D ** -0.5)
    qc, kc, vc = (t.cuda().requires_grad_(True) for t in (q, k, v))
    out = prefill.window_attention(qc, kc, vc, window=window, num_sinks=sinks, scale=scale)
    R.check_out(out.detach(), O, A, (S, window, sinks))
    check(torch.autograd.grad(out, (qc, kc, vc), do.cuda()), grads, (S, window, sinks))
    _, l2 = prefill.window_forward(qc.detach(), kc.detach(), vc.detach(), window=window, num_sinks=sinks, scale=scale,
                                   return_lse=True)
    assert ((l2.double().cpu() - lse).abs() <= 2.0 ** -12 + 2.0 ** -22 * lse.abs()).all()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("S", [1, 2, 63, 64, 65, 127, 128, 129, 200, 333, 513])
@pytest.mark.parametrize("window,sinks", [(1, 0), (37, 3), (128, 64), (1000, 0)])
def test_lengths(D, S, window, sinks):
    run(1, 2, 1, S, D, window, sinks, seed=S)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("window,sinks", [(1, 1), (64, 1), (65, 130), (200, 70), (255, 400), (256, 128), (300, 0)])
def test_windows(D, window, sinks):
    run(2, 4, 2, 640, D, window, sinks)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,Hkv", [(1, 1), (3, 1), (8, 8), (8, 2), (6, 2), (16, 2)])
def test_heads(D, H, Hkv):
    run(1, H, Hkv, 257, D, 90, 5, scale=0.2, bshd=False)


def test_long_sinks_range():
    """The sinks' key tile sees every query tile (more pairs than the window's tiles by far)."""
    run(1, 4, 1, 4200, 64, 50, 2)
    run(1, 4, 1, 4200, 128, 50, 2)


def test_directional_differences():
    """The kernel's gradients against central differences of the 64-bit forward."""
    q, k, v, do = inputs(1, 4, 2, 150, 64, seed=4)
    qc, kc, vc = (t.cuda().requires_grad_(True) for t in (q, k, v))
    out = prefill.window_attention(qc, kc, vc, window=40, num_sinks=2)
    grads = [t.double().cpu() for t in torch.autograd.grad(out, (qc, kc, vc), do.cuda())]
    _, pairs, _ = formulas(q, k, v, do, 40, 2, 0.125)
    g = torch.Generator().manual_seed(5)
    for i in range(3):
        d = torch.randn(grads[i].shape, generator=g, dtype=torch.float64)
        vals = []
        for sgn in (1, -1):
            a = [t.double() for t in (q, k, v)]
            a[i] = a[i] + sgn * 1e-5 * d
            (O, _), _, _ = formulas(a[0], a[1], a[2], do, 40, 2, 0.125)
            vals.append((O * do.double()).sum())
        diff = (vals[0] - vals[1]) / 2e-5
        assert abs((grads[i] * d).sum() - diff) <= (pairs[i][1] * d.abs()).sum() + 1e-5 * diff.abs()


def test_rows_past_the_end_do_not_leak_into_the_next_head():
    """S that fills no tile: every head's gradients are those of the head alone."""
    for D in (64, 128):
        q, k, v, do = (t.cuda() for t in inputs(2, 4, 4, 70, D, seed=6))
        out, lse = prefill.window_forward(q, k, v, window=30, num_sinks=1, return_lse=True)
        full = prefill.window_backward(q, k, v, out, do, lse, window=30, num_sinks=1)
        for b in range(2):
            for h in range(4):
                s = (slice(b, b + 1), slice(h, h + 1))
                o1, l1 = prefill.window_forward(q[s], k[s], v[s], window=30, num_sinks=1, return_lse=True)
                one = prefill.window_backward(q[s], k[s], v[s], o1, do[s], l1, window=30, num_sinks=1)
                assert torch.equal(o1, out[s])
                for a, c in zip(one, full):
                    assert torch.equal(a, c[s])


def test_broadcast_and_odd_views():
    """Expanded keys (gradient summed by autograd), a misaligned view, an expanded upstream gradient."""
    q, k, v, _ = (t.cuda() for t in inputs(1, 4, 1, 100, 64, seed=7))
    ke, ve = k.clone().requires_grad_(True), v.clone().requires_grad_(True)
    a = prefill.window_attention(q, ke.expand(1, 4, 100, 64), ve.expand(1, 4, 100, 64), window=20, num_sinks=1)
    k1, v1 = k.clone().requires_grad_(True), v.clone().requires_grad_(True)
    b = prefill.window_attention(q, k1, v1, window=20, num_sinks=1)
    assert torch.equal(a, b)
    ones = torch.ones((1, 1, 1, 1), dtype=torch.bfloat16, device="cuda").expand(1, 4, 100, 64)
    ga = torch.autograd.grad(a, (ke, ve), ones)
    gb = torch.autograd.grad(b, (k1, v1), ones.contiguous())
    for x, y in zip(ga, gb):  # four heads' gradients rounded before or after their sum
        assert ((x - y).float().abs() <= 2.0 ** -5 * y.float().abs().max()).all()
    flat = torch.zeros(q.numel() + 3, dtype=torch.bfloat16, device="cuda")
    odd = flat[3:].view(1, 100, 4, 64).transpose(1, 2)
    odd.copy_(q)
    assert odd.data_ptr() % 16
    assert torch.equal(prefill.window_forward(odd, k, v, window=20, num_sinks=1), b)


def test_graph_capture():
    """Forward and backward in one graph.  (torch itself refuses to capture a backward pass while an eager
    graph of the same leaf tensors is alive, whatever the operator: the eager one is released first.)"""
    q, k, v, do = (t.cuda() for t in inputs(1, 4, 2, 300, 128, seed=8))
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    eager = prefill.window_attention(*leaves, window=64, num_sinks=4)
    ref = torch.autograd.grad(eager, leaves, do)
    eager = eager.detach()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = prefill.window_attention(*leaves, window=64, num_sinks=4)
        grads = torch.autograd.grad(out, leaves, do)
    for _ in range(2):
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
        assert torch.equal(grads[1], ref[1]) and torch.equal(grads[2], ref[2])
        assert (grads[0] - ref[0]).float().abs().max() <= 2.0 ** -7 * ref[0].float().abs().max()


def test_two_streams_at_once():
    q, k, v, do = (t.cuda() for t in inputs(1, 4, 2, 700, 128, seed=9))
    out, lse = prefill.window_forward(q, k, v, window=100, return_lse=True)
    ref = prefill.window_backward(q, k, v, out, do, lse, window=100)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    res = [prefill.window_backward(q, k, v, out, do, lse, window=100, stream=s) for s in streams for _ in range(3)]
    torch.cuda.synchronize()
    for r in res:
        assert torch.equal(r[1], ref[1]) and torch.equal(r[2], ref[2])
        assert (r[0] - ref[0]).float().abs().max() <= 2.0 ** -7 * ref[0].float().abs().max()


def test_attention_interface():
    q, k, v, do = (t.cuda() for t in inputs(1, 4, 2, 130, 64, seed=10))
    m = prefill.WindowMask(window=33, num_sinks=2)
    out, _ = prefill.abkv_attention_forward(None, q, k, v, m, scaling=0.2)
    assert torch.equal(out.transpose(1, 2), prefill.window_forward(q, k, v, window=33, num_sinks=2, scale=0.2))
    qg = q.clone().requires_grad_(True)
    out2, _ = prefill.abkv_attention_forward(None, qg, k, v, m, scaling=0.2)
    assert torch.equal(out, out2) and torch.autograd.grad(out2.sum(), qg)[0].abs().sum() > 0


def test_refusals():
    q, k, v, do = (t.cuda() for t in inputs(1, 4, 2, 40, 64, seed=11))
    for kw in (dict(window=0), dict(window=-3), dict(window=4, num_sinks=-1)):
        with pytest.raises(ValueError, match="window"):
            prefill.window_attention(q, k, v, **kw)
    with pytest.raises(TypeError, match="bf16"):
        prefill.window_attention(q.float(), k, v, window=4)
    with pytest.raises(ValueError, match="matching"):
        prefill.window_attention(q, k[:, :, :30], v, window=4)
    with pytest.raises(ValueError, match="divide"):
        prefill.window_attention(q[:, :3], k, v, window=4)
    with pytest.raises(RuntimeError):
        prefill.window_attention(*(torch.zeros((1, 1, 8, 96), dtype=torch.bfloat16, device="cuda"),) * 3, window=4)
    with pytest.raises(ValueError, match="lse"):
        prefill.window_backward(q, k, v, q, do, torch.zeros((1, 4, 39), device="cuda"), window=4)
    with pytest.raises(RuntimeError):
        prefill.window_forward(q, k, v, window=4, scale=-1.0, workspace=Workspace("cuda:0"))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("S,window,sinks,alone", [(1, 5, 0, 1), (1, 5, 3, 1), (150, 1, 0, 150), (150, 1, 2, 1), (150, 40, 0, 1),
                                                  (700, 600, 4, 1)])
def test_rows_that_see_one_key_have_no_score_gradient(D, S, window, sinks, alone):
    """Their weight is 1 whatever the score, so dq is exactly 0 there, and dk where no other row sees the key."""
    g = torch.Generator().manual_seed(S + D)
    q, k, v, do = (torch.randn((2, h, S, D), generator=g).bfloat16().cuda() for h in (4, 2, 2, 4))
    for t in (q, k, v):
        t.requires_grad_()
    out = prefill.window_attention(q, k, v, window=window, num_sinks=sinks)
    dq, dk, dv = torch.autograd.grad(out, (q, k, v), do)
    assert torch.equal(out[:, :, :alone], v.repeat_interleave(2, 1)[:, :, :alone])
    assert (dq[:, :, :alone] == 0).all() and (alone == S or (dq[:, :, alone:] != 0).any())
    if alone == S:
        assert (dk == 0).all()
        # each key has its own row's gradient, summed over the two heads that share it
        want = do.double().view(2, 2, 2, S, D).sum(2)
        assert (dv.double() - want).abs().le(2.0 ** -8 * want.abs() + 1e-30).all()


def test_gradients_are_not_differentiable_again():
    """Under create_graph the gradients come out, and a second derivative is refused rather than left out."""
    g = torch.Generator().manual_seed(2)
    q, k, v, do = (torch.randn((1, h, 70, 64), generator=g).bfloat16().cuda() for h in (4, 2, 2, 4))
    for t in (q, k, v):
        t.requires_grad_()
    plain = torch.autograd.grad(prefill.window_attention(q, k, v, window=9), (q, k, v), do)
    again = torch.autograd.grad(prefill.window_attention(q, k, v, window=9), (q, k, v), do, create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(plain, again))
    with pytest.raises(RuntimeError):  # (torch: of a dout without a gradient of its own the result has none either)
        torch.autograd.grad(again[0].float().sum(), q)
    do.requires_grad_()
    again = torch.autograd.grad(prefill.window_attention(q, k, v, window=9), (q, k, v), do, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        again[0].float().sum().backward()
