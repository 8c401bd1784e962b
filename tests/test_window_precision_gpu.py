"""What the training attention keeps beside its bf16 outputs, on the GPU: the forward's low mantissa bits, the second
bf16 part of dS where rows see few keys, and results that repeat bit for bit.

Bounds (u = 2^-8, e = 2^-12 as in bounded_ref):
* low bits: eight more bits of the output's mantissa, a step of 2^-15 of its magnitude; rounded, or one step short where
  the last rounding would carry: |error| <= 2^-15 |out| beside the 32-bit sums.
* gradients from an output of 64 bits in those 16 mantissa bits: Di = sum dO O within 2^-15 sum |dO| |O|, dP within
  D 2^-23 <= 2^-16 of sum |dO| |V|, P within e of itself, dS in two bf16 parts within u^2 of itself, in one within u:
  d = u^2 |dS| (u |dS| in one part) + P (e (|dP| + |Di|) + 2^-16 sum |dO| |V| + 2^-15 sum |dO| |O|);
  dQ and dK multiply it out, each rounded once more: scale d |K| + u |dQ|, scale d^T |Q| + u |dK|.
Without the low bits, or with dS in one part, errors were 4 to 8 times this bound in a 64-bit emulation."""
import pytest
import torch

import bounded_ref as R
from abridgekv_b200 import prefill

pytestmark = pytest.mark.gpu
U, E = R.U16, R.U32


def bf16(shape, g):
    return torch.randn(shape, generator=g).to(torch.bfloat16)


def split(x):
    """x (64 bits) -> bf16 and the int8 of the next mantissa bits, as window_forward returns them."""
    hi = x.float().bfloat16()
    d = x.float().view(torch.int32) - hi.float().view(torch.int32)
    return hi, ((d.clamp(max=32639) + 128) >> 8).to(torch.int8)


def joined(out, low):
    return (out.float().contiguous().view(torch.int32) + (low.int() << 8)).view(torch.float32)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,H,Hkv,S,window,sinks", [(1, 2, 1, 70, 9, 0), (2, 4, 2, 333, 50, 3), (1, 3, 3, 200, 200, 0)])
def test_low_bits_of_the_output(D, B, H, Hkv, S, window, sinks):
    """With q = 0 every weight is 1: the output is a mean of V rows, whose low bits the bf16 output does not have."""
    g = torch.Generator().manual_seed(S + D)
    k, v = bf16((B, Hkv, S, D), g), bf16((B, Hkv, S, D), g)
    out, low = prefill.window_forward(torch.zeros((B, H, S, D), dtype=torch.bfloat16, device="cuda"), k.cuda(), v.cuda(),
                                      window=window, num_sinks=sinks, return_low=True)
    vis = R.visible(list(range(S)), S, window, sinks).double()
    P = vis / vis.sum(-1, keepdim=True)
    V = v.double().repeat_interleave(H // Hkv, 1)
    want, size = P @ V, P @ V.abs()
    got = joined(out.cpu(), low.cpu()).double()
    assert ((got - want).abs() <= 2.0 ** -15 * want.abs() + S * 2.0 ** -23 * size).all()
    assert (low != 0).float().mean() > 0.5  # the bf16 output alone is not that near


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,H,Hkv,S,window,sinks", [
    (1, 4, 2, 300, 130, 4), (2, 2, 2, 140, 1000, 0), (1, 2, 1, 1100, 500, 12),  # no row sees more than 512 keys: two parts
    (1, 2, 1, 900, 900, 0), (1, 2, 2, 1100, 700, 3), (1, 2, 1, 700, 20, 600),   # some do: one part for all rows
])
def test_gradients_from_an_output_with_its_low_bits(D, B, H, Hkv, S, window, sinks):
    g = torch.Generator().manual_seed(S + D)
    q, k, v, do = (bf16((B, h, S, D), g) for h in (H, Hkv, Hkv, H))
    scale, G = D ** -0.5, H // Hkv
    Q, dO = q.double(), do.double()
    K, V = (t.double().repeat_interleave(G, 1) for t in (k, v))
    vis = R.visible(list(range(S)), S, window, sinks)
    x = (Q @ K.transpose(2, 3) * scale).masked_fill(~vis, float("-inf"))
    lse, P = x.logsumexp(-1), torch.softmax(x, -1)
    O, dP = P @ V, dO @ V.transpose(2, 3)
    Di = (dO * O).sum(-1, keepdim=True)
    dS = P * (dP - Di)
    d = (U * U if min(S, window + sinks) <= 512 else U) * dS.abs() + P * (
        E * (dP.abs() + Di.abs()) + 2.0 ** -16 * (dO.abs() @ V.abs().transpose(2, 3)) +
        2.0 ** -15 * (dO.abs() * O.abs()).sum(-1, keepdim=True))

    def heads(t):
        return t.reshape(B, Hkv, G, S, D).sum(2)

    dq, dk = scale * dS @ K, heads(scale * dS.transpose(2, 3) @ Q)
    bq = scale * d @ K.abs() + U * dq.abs() + 1e-30
    bk = heads(scale * d.transpose(2, 3) @ Q.abs()) + U * dk.abs() + 1e-30
    out, low = (t.cuda() for t in split(O))
    got = prefill.window_backward(q.cuda(), k.cuda(), v.cuda(), out, do.cuda(), lse.float().cuda(), window=window,
                                  num_sinks=sinks, low=low)
    for name, t, ref, bound in (("dq", got[0], dq, bq), ("dk", got[1], dk, bk)):
        worst = ((t.double().cpu() - ref).abs() / bound).amax((0, 1, 3))
        assert worst.max() <= 1, (name, float(worst.max()), int(worst.argmax()))
    if min(S, window + sinks) <= 512:  # the bound is near enough to see that the low bits are used
        bare = prefill.window_backward(q.cuda(), k.cuda(), v.cuda(), out, do.cuda(), lse.float().cuda(), window=window,
                                       num_sinks=sinks)
        assert ((bare[0].double().cpu() - dq).abs() > bq).any()


def step(B, H, Hkv, S, D, window, sinks, seed=0):
    g = torch.Generator().manual_seed(seed)
    leaves = [bf16((B, h, S, D), g).cuda().requires_grad_(True) for h in (H, Hkv, Hkv)]
    do = bf16((B, H, S, D), g).cuda()

    def run():
        out = prefill.window_attention(*leaves, window=window, num_sinks=sinks)
        return [out.detach(), *torch.autograd.grad(out, leaves, do)]

    return run


# more query tiles x heads than SMs (several items a CTA), short (clusters for dK / dV), sinks' tiles of their own launch
REPEATS = [(2, 16, 4, 1300, 128, 300, 4), (1, 8, 2, 333, 64, 128, 1), (1, 8, 2, 4200, 64, 50, 2), (2, 8, 8, 700, 128, 1000, 0)]


@pytest.mark.parametrize("shape", REPEATS)
def test_gradients_repeat_bit_for_bit(shape):
    run = step(*shape)
    first = run()
    for _ in range(60):
        assert all(torch.equal(a, b) for a, b in zip(run(), first))


def test_gradients_of_a_graph_and_of_two_streams_are_the_same_bits():
    runs = [step(1, 16, 4, 1500, 128, 200, 3, seed=i) for i in range(2)]
    first = [r() for r in runs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in runs]
    for _ in range(5):
        got = []
        for r, s in zip(runs * 2, streams * 2):
            with torch.cuda.stream(s):
                got.append(r())
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for i, t in enumerate(got) for a, b in zip(t, first[i % 2]))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = runs[0]()
    for _ in range(5):
        for t in out:
            t.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, first[0]))
