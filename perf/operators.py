"""The operators of a bounded KV cache as a user calls them: attention with a sliding window and
sinks (one token over the paged cache, ragged prompt rows over the paged cache, training with its
gradients) and eviction by accumulated attention weight (weights of decode steps, weights of prompt
rows, the eviction itself).

``own`` False runs the plain form (elementary torch operations in 32 bits), True the framework's
entry points.  Both take what ``prepare`` makes."""
import math

import numpy as np
import torch

own = False

DEV = "cuda"


# ---------------------------------------------------------------- cases
def listed():
    return [
        # one sequence, one layer of a model: the latency of a single layer call (the default head layout)
        dict(name="decode_window_one", kind="decode_window", L=1, B=1, Hq=32, Hkv=8, D=128, page=16, lo=4097, hi=4097,
             window=1024, sinks=4),
        # a served batch, several layers in one launch, ragged lengths, pages behind the window already freed
        dict(name="decode_window_batch", kind="decode_window", L=8, B=32, Hq=32, Hkv=8, D=128, page=16, lo=1801,
             hi=9973, window=4096, sinks=4),
        # a chunk of a prompt beside two short requests (chunked prefill), FlashAttention page layout
        dict(name="prompt_window_chunk", kind="prompt_window", R=3, Hq=32, Hkv=8, page=16, layout=1, qlo=37, qhi=300,
             hist=517, window=256, sinks=4),
        # whole prompts of 8K tokens
        dict(name="prompt_window_long", kind="prompt_window", R=2, Hq=32, Hkv=8, page=16, layout=0, qlo=8191, qhi=8191,
             hist=0, window=2048, sinks=4),
        # a small training step: head size 64, a length that fills no tile
        dict(name="train_window_small", kind="train_window", B=1, H=8, Hkv=2, S=333, D=64, window=128, sinks=1),
        # a training step of one layer at 4K tokens
        dict(name="train_window_4k", kind="train_window", B=2, H=32, Hkv=8, S=4096, D=128, window=1024, sinks=4),
        # one sequence whose cache is watched head by head
        dict(name="decode_weighted_one", kind="decode_weighted", L=1, B=1, Hq=32, Hkv=8, D=128, page=16, lo=1531,
             hi=1531, units=8),
        # a served batch, weights summed over all heads, ragged lengths
        dict(name="decode_weighted_batch", kind="decode_weighted", L=4, B=32, Hq=32, Hkv=8, D=128, page=16, lo=4003,
             hi=8190, units=1),
        # the last 32 prompt rows vote on an 8K prompt (observation window), before its first eviction
        dict(name="prompt_weights_observe", kind="prompt_weights", R=4, Hq=32, Hkv=8, page=16, layout=0, qlo=64, qhi=64,
             hist=8001, observe=32, window=0, sinks=0, units=8),
        # every row of a 4K prompt votes
        dict(name="prompt_weights_all", kind="prompt_weights", R=2, Hq=32, Hkv=8, page=16, layout=0, qlo=4001,
             qhi=4096, hist=0, observe=0, window=0, sinks=0, units=8),
        # one sequence goes back to its budget, each KV head its own rows
        dict(name="evict_one", kind="evict", L=1, B=1, Hkv=8, D=128, page=16, lo=1311, hi=1311, budget=1024, sinks=4,
             recent=64, units=8),
        # a batch after its prompts: half of the rows go, all heads keep the same rows
        dict(name="evict_batch", kind="evict", L=4, B=16, Hkv=8, D=128, page=16, lo=5003, hi=8190, budget=4096,
             sinks=4, recent=256, units=1),
    ]


def _logint(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["decode_window", "prompt_window", "train_window", "decode_weighted", "prompt_weights", "evict"])
    Hkv = rng.choice([1, 2, 4, 8])
    G = rng.randint(1, 8)
    page = rng.choice([16, 32, 64])
    if kind in ("decode_window", "decode_weighted"):
        hi = _logint(rng, 1, 20000)
        L, B = rng.randint(1, 3), _logint(rng, 1, 24)
        c = dict(kind=kind, L=L, B=B, Hq=Hkv * G, Hkv=Hkv, D=rng.choice([64, 128]), page=page,
                 lo=rng.randint(0, hi), hi=hi)
        if kind == "decode_window":
            c.update(window=_logint(rng, 1, 6000), sinks=rng.choice([0, 1, 4, rng.randint(5, 100)]))
        else:
            c.update(units=rng.choice([1, Hkv]))
            c["hi"] = min(hi, 12000)
            c["lo"] = min(c["lo"], c["hi"])
        return c
    if kind in ("prompt_window", "prompt_weights"):
        qhi = _logint(rng, 1, 3000)
        c = dict(kind=kind, R=rng.randint(1, 4), Hq=Hkv * G, Hkv=Hkv, page=page, layout=rng.choice([0, 1]),
                 qlo=rng.randint(1, qhi), qhi=qhi, hist=rng.choice([0, _logint(rng, 1, 4000)]),
                 window=_logint(rng, 1, 4000), sinks=rng.choice([0, 1, 4, rng.randint(5, 200)]))
        if kind == "prompt_weights":
            c.update(observe=rng.choice([0, _logint(rng, 1, 200)]), units=rng.choice([1, Hkv]))
            if rng.random() < 0.5:
                c.update(window=0, sinks=0)
        return c
    if kind == "train_window":
        S = _logint(rng, 1, 3000)
        return dict(kind=kind, B=rng.randint(1, 2), H=Hkv * min(G, 4), Hkv=Hkv, S=S, D=rng.choice([64, 128]),
                    window=_logint(rng, 1, 2048), sinks=rng.choice([0, 1, 4, rng.randint(5, 200)]))
    hi = _logint(rng, 2, 8000)
    sinks, recent = rng.randint(0, 8), rng.randint(0, 300)
    return dict(kind=kind, L=rng.randint(1, 2), B=_logint(rng, 1, 12), Hkv=Hkv, D=rng.choice([64, 128]), page=page,
                lo=rng.randint(0, hi), hi=hi, budget=sinks + recent + _logint(rng, 1, hi), sinks=sinks, recent=recent,
                units=rng.choice([1, Hkv]))


def _spread(n, lo, hi):
    """n lengths from lo to hi (the first is hi), the same for every seed."""
    if n == 1:
        return [hi]
    return [hi - (hi - lo) * ((5 * i) % n) // (n - 1) for i in range(n)]


def _lens(c):
    if "R" in c:
        q = _spread(c["R"], c["qlo"], c["qhi"])
        return q, [x + c["hist"] * (i + 1) // c["R"] for i, x in enumerate(q)]
    return _spread(c["B"], c["lo"], c["hi"])


# ---------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed) * 7919 + 17)


def _randn(g, shape, scale=1.0):
    return (torch.randn(shape, generator=g, device=DEV, dtype=torch.float32) * scale).to(torch.bfloat16)


def _cache(g, nb, c, layout=0):
    D = c.get("D", 128)
    shape = (nb, 2, c["page"], c["Hkv"], D) if layout == 0 else (2, nb, c["page"], c["Hkv"], D)
    out = torch.empty(shape, device=DEV, dtype=torch.bfloat16)
    flat = out.view(-1)
    step = 1 << 28
    for i in range(0, flat.numel(), step):
        n = min(step, flat.numel() - i)
        flat[i:i + n] = _randn(g, (n,))
    return out


def _tables(seed, lens, page, first=None):
    """Shuffled pages of each sequence (page 0 is the null block).  first[b] (optional) is the set of
    live page slots; the others were freed and name the null block.  -> (table, number of pages)"""
    rng = np.random.default_rng(int(seed) + 5)
    counts = [(n + page - 1) // page for n in lens]
    live = [np.arange(k) if first is None else first[b] for b, k in enumerate(counts)]
    total = int(sum(len(x) for x in live))
    ids = 1 + rng.permutation(total)
    table = np.zeros((len(lens), max(1, max(counts))), dtype=np.int32)
    at = 0
    for b, slots in enumerate(live):
        table[b, slots] = ids[at:at + len(slots)]
        at += len(slots)
    return torch.from_numpy(table).to(DEV), total + 1


def _visible_span(n, window, sinks):
    """Rows the token at position n - 1 sees: [0, s) and [w, n)."""
    if window <= 0:
        return 0, 0
    w = max(0, n - window)
    return min(sinks, w), w


def prepare(case, seed):
    c, g = case, _gen(seed)
    k = c["kind"]
    st = dict(c=c)
    if k in ("decode_window", "decode_weighted"):
        lens = _lens(c)
        win, sinks = c.get("window", 0), c.get("sinks", 0)
        live = []
        for n in lens:
            s, w = _visible_span(n, win, sinks)
            slots = set(range(0, (s + c["page"] - 1) // c["page"])) | set(
                range(w // c["page"], (n + c["page"] - 1) // c["page"]))
            live.append(np.array(sorted(slots), dtype=np.int64))
        st.update(q=[], kv=[], bt=[], lens=lens)
        sl = torch.tensor(lens, dtype=torch.int32, device=DEV)
        st["sl"] = [sl] * c["L"]
        for layer in range(c["L"]):
            bt, nb = _tables(seed * 31 + layer, lens, c["page"], live)
            st["bt"].append(bt)
            st["kv"].append(_cache(g, nb, c))
            st["q"].append(_randn(g, (c["B"], c["Hq"], c["D"])))
        if k == "decode_weighted":
            cap = st["bt"][0].shape[1] * c["page"]
            st["w"] = [torch.rand((c["B"], c["units"], cap), generator=g, device=DEV) for _ in range(c["L"])]
    elif k in ("prompt_window", "prompt_weights"):
        q, lens = _lens(c)
        bt, nb = _tables(seed, lens, c["page"])
        T = sum(q)
        st.update(qlens=q, lens=lens, bt=bt, kv=_cache(g, nb, c, c["layout"]), q=_randn(g, (T, c["Hq"], 128)),
                  sl=torch.tensor(lens, dtype=torch.int32, device=DEV),
                  qs=torch.tensor(np.concatenate([[0], np.cumsum(q)]), dtype=torch.int32, device=DEV))
        if k == "prompt_weights":
            # the log-sum-exp that the attention of these rows left behind
            st["lse"] = _prompt_plain(st)[1]
            st["w"] = torch.rand((c["R"], c["units"], bt.shape[1] * c["page"]), generator=g, device=DEV)
    elif k == "train_window":
        # activations as the model holds them: [B, S, heads, D], viewed as [B, heads, S, D]
        for name, h in (("q", c["H"]), ("k", c["Hkv"]), ("v", c["Hkv"])):
            st[name] = _randn(g, (c["B"], c["S"], h, c["D"])).transpose(1, 2).requires_grad_(True)
        st["do"] = _randn(g, (c["B"], c["S"], c["H"], c["D"])).transpose(1, 2)
    else:
        lens = _lens(c)
        m = [min(n, c["budget"]) for n in lens]
        both = lens + m  # source pages, then the pages that the kept rows move to
        bt, nb = _tables(seed, both, c["page"])
        st.update(lens=lens, bt=[bt[:c["B"]].contiguous()] * c["L"], sl=[torch.tensor(lens, dtype=torch.int32,
                                                                                      device=DEV)] * c["L"],
                  dst=[bt[c["B"]:].contiguous()] * c["L"], kv=[_cache(g, nb, c) for _ in range(c["L"])], w=[])
        cap = bt.shape[1] * c["page"]
        for _ in range(c["L"]):
            # sums of attention weights: a few heavy rows, a long light tail
            u = torch.rand((c["B"], c["units"], cap), generator=g, device=DEV)
            st["w"].append(torch.exp(-6.0 * u) * u)
    return st


# ---------------------------------------------------------------- plain forms
def _rows(kv, layout, table, rows, page, dtype):
    """K and V rows [n, Hkv, D] of one sequence through its block table."""
    pages = table[rows // page].long()
    off = rows % page
    if layout == 0:
        return kv[pages, 0, off].to(dtype), kv[pages, 1, off].to(dtype)
    return kv[0][pages, off].to(dtype), kv[1][pages, off].to(dtype)


def _decode_plain(st, weighted):
    c = st["c"]
    G, scale = c["Hq"] // c["Hkv"], 1.0 / math.sqrt(c["D"])
    outs, ws = [], []
    for layer in range(c["L"]):
        out = torch.zeros((c["B"], c["Hq"], c["D"]), device=DEV)
        w = st["w"][layer].clone() if weighted else None
        for b, n in enumerate(st["lens"]):
            if n == 0:
                continue
            s, lo = _visible_span(n, c.get("window", 0), c.get("sinks", 0))
            rows = torch.cat([torch.arange(s, device=DEV), torch.arange(lo, n, device=DEV)])
            K, V = _rows(st["kv"][layer], 0, st["bt"][layer][b], rows, c["page"], torch.float32)
            q = st["q"][layer][b].float().view(c["Hkv"], G, c["D"])
            x = torch.matmul(q, K.permute(1, 2, 0)) * scale
            x = x - x.amax(-1, keepdim=True)
            e = torch.exp(x)
            p = e / e.sum(-1, keepdim=True)
            out[b] = torch.matmul(p, V.permute(1, 0, 2)).reshape(c["Hq"], c["D"])
            if weighted:
                add = p.sum(1)
                w[b, :, :n] += add if c["units"] > 1 or c["Hkv"] == 1 else add.sum(0, keepdim=True)
        outs.append(out.to(torch.bfloat16))
        ws.append(w)
    return outs, ws


def _mask(pos, n, window, sinks):
    j = torch.arange(n, device=DEV)
    vis = j[None, :] <= pos[:, None]
    if window > 0:
        vis = vis & ((j[None, :] > pos[:, None] - window) | (j[None, :] < sinks))
    return vis


def _prompt_plain(st):
    c = st["c"]
    G, scale = c["Hq"] // c["Hkv"], 1.0 / math.sqrt(128)
    out = torch.empty_like(st["q"])
    lse = torch.empty(st["q"].shape[:2], device=DEV)
    t0 = 0
    for r, (nq, n) in enumerate(zip(st["qlens"], st["lens"])):
        K, V = _rows(st["kv"], c["layout"], st["bt"][r], torch.arange(n, device=DEV), c["page"], torch.float32)
        for a in range(0, nq, 1024):
            e1 = min(a + 1024, nq)
            pos = torch.arange(n - nq + a, n - nq + e1, device=DEV)
            hid = ~_mask(pos, n, c["window"], c["sinks"])
            for h in range(c["Hkv"]):
                q = st["q"][t0 + a:t0 + e1, h * G:(h + 1) * G].float().transpose(0, 1)
                x = (torch.matmul(q, K[:, h].t()) * scale).masked_fill(hid, float("-inf"))
                m = x.amax(-1, keepdim=True)
                e = torch.exp(x - m)
                z = e.sum(-1, keepdim=True)
                out[t0 + a:t0 + e1, h * G:(h + 1) * G] = torch.matmul(e / z, V[:, h]).transpose(0, 1).to(out.dtype)
                lse[t0 + a:t0 + e1, h * G:(h + 1) * G] = (m + torch.log(z)).squeeze(-1).t()
        t0 += nq
    return out, lse


def _prompt_weights_plain(st):
    c = st["c"]
    G, scale = c["Hq"] // c["Hkv"], 1.0 / math.sqrt(128)
    w = st["w"].clone()
    t0 = 0
    for r, (nq, n) in enumerate(zip(st["qlens"], st["lens"])):
        K, _ = _rows(st["kv"], c["layout"], st["bt"][r], torch.arange(n, device=DEV), c["page"], torch.float32)
        first = max(0, nq - c["observe"]) if c["observe"] else 0
        for a in range(first, nq, 1024):
            e1 = min(a + 1024, nq)
            pos = torch.arange(n - nq + a, n - nq + e1, device=DEV)
            vis = _mask(pos, n, c["window"], c["sinks"])
            for h in range(c["Hkv"]):
                q = st["q"][t0 + a:t0 + e1, h * G:(h + 1) * G].float().transpose(0, 1)
                x = torch.matmul(q, K[:, h].t()) * scale - st["lse"][t0 + a:t0 + e1, h * G:(h + 1) * G].t()[..., None]
                p = torch.exp(x.masked_fill(~vis, float("-inf")))
                w[r, h if c["units"] > 1 else 0, :n] += p.sum((0, 1))
        t0 += nq
    return w


def _train(st, dtype):
    """out, dq, dk, dv by their formulas, head group by head group."""
    c = st["c"]
    G, scale = c["H"] // c["Hkv"], 1.0 / math.sqrt(c["D"])
    q, k, v, do = (st[x].detach() for x in ("q", "k", "v", "do"))
    out, dq, dk, dv = (torch.empty_like(t, dtype=torch.bfloat16 if dtype == torch.float32 else dtype)
                       for t in (q, q, k, v))
    hid = ~_mask(torch.arange(c["S"], device=DEV), c["S"], c["window"], c["sinks"])
    for b in range(c["B"]):
        for h in range(c["Hkv"]):
            hs = slice(h * G, (h + 1) * G)
            Q, K, V, dO = q[b, hs].to(dtype), k[b, h].to(dtype), v[b, h].to(dtype), do[b, hs].to(dtype)
            x = (torch.matmul(Q, K.t()) * scale).masked_fill(hid, float("-inf"))
            e = torch.exp(x - x.amax(-1, keepdim=True))
            P = e / e.sum(-1, keepdim=True)
            del x, e
            O = torch.matmul(P, V)
            dP = torch.matmul(dO, V.t())
            dS = P * (dP - (dP * P).sum(-1, keepdim=True))
            out[b, hs] = O.to(out.dtype)
            dq[b, hs] = (torch.matmul(dS, K) * scale).to(out.dtype)
            dk[b, h] = (torch.matmul(dS.transpose(1, 2), Q).sum(0) * scale).to(out.dtype)
            dv[b, h] = torch.matmul(P.transpose(1, 2), dO).sum(0).to(out.dtype)
    return out, dq, dk, dv


def _evict_plain(st):
    c = st["c"]
    new_lens, ws, keeps = [], [], []
    for layer in range(c["L"]):
        kv, w = st["kv"][layer], st["w"][layer]
        m, W = c["budget"], torch.zeros_like(w)
        keep = torch.full((c["B"], c["units"], m), -1, dtype=torch.int32, device=DEV)
        new = torch.zeros(c["B"], dtype=torch.int32, device=DEV)
        for b, n in enumerate(st["lens"]):
            k = min(n, m)
            new[b] = k
            for u in range(c["units"]):
                if n <= m:
                    rows = torch.arange(n, device=DEV)
                else:
                    mid = w[b, u, c["sinks"]:n - c["recent"]]
                    top = torch.sort(mid, descending=True, stable=True)[1][:m - c["sinks"] - c["recent"]]
                    rows = torch.cat([torch.arange(c["sinks"], device=DEV), c["sinks"] + torch.sort(top)[0],
                                      torch.arange(n - c["recent"], n, device=DEV)])
                keep[b, u, :k] = rows.int()
                W[b, u, :k] = w[b, u, rows]
                j = torch.arange(k, device=DEV)
                src, dst = st["bt"][layer][b][rows // c["page"]].long(), st["dst"][layer][b][j // c["page"]].long()
                if c["units"] == 1:
                    kv[dst, :, j % c["page"]] = kv[src, :, rows % c["page"]]
                else:
                    kv[dst, :, j % c["page"], u] = kv[src, :, rows % c["page"], u]
        new_lens.append(new)
        ws.append(W)
        keeps.append(keep)
    return dict(kv=st["kv"], new_lens=new_lens, weights=ws, keep=keeps)


def run(state):
    c = state["c"]
    k = c["kind"]
    if not own:
        with torch.no_grad():
            if k == "decode_window":
                return _decode_plain(state, False)[0]
            if k == "decode_weighted":
                return _decode_plain(state, True)
            if k == "prompt_window":
                return _prompt_plain(state)
            if k == "prompt_weights":
                return _prompt_weights_plain(state)
            if k == "train_window":
                return _train(state, torch.float32)
            return _evict_plain(state)
    from abridgekv_b200 import codestep, compaction, decode, prefill
    if k == "decode_window":
        return decode.paged_decode_window(state["q"], state["kv"], state["bt"], state["sl"], window=c["window"],
                                          num_sinks=c["sinks"])
    if k == "decode_weighted":
        w = [x.clone() for x in state["w"]]
        return decode.paged_decode_weighted(state["q"], state["kv"], state["bt"], state["sl"], w), w
    if k == "prompt_window":
        return codestep.paged_prefill_window(state["q"], state["kv"], state["bt"], state["sl"], state["qs"],
                                             max_query_len=c["qhi"], num_kv_heads=c["Hkv"], window=c["window"],
                                             num_sinks=c["sinks"], return_lse=True)
    if k == "prompt_weights":
        w = state["w"].clone()
        return codestep.paged_prompt_weights(state["q"], state["lse"], state["kv"], state["bt"], state["sl"],
                                             state["qs"], w, num_kv_heads=c["Hkv"], max_query_len=c["qhi"],
                                             observe=c["observe"] or None, window=c["window"] or None,
                                             num_sinks=c["sinks"])
    if k == "train_window":
        out = prefill.window_attention(state["q"], state["k"], state["v"], window=c["window"], num_sinks=c["sinks"])
        return (out.detach(), *torch.autograd.grad(out, (state["q"], state["k"], state["v"]), state["do"]))
    res = compaction.evict_by_weight(state["kv"], state["bt"], state["sl"], state["w"], budget=c["budget"],
                                     num_sinks=c["sinks"], num_recent=c["recent"], dst_block_tables=state["dst"],
                                     return_keep=True)
    return dict(kv=state["kv"], new_lens=res.seq_lens, weights=res.weights, keep=res.keep)


# ---------------------------------------------------------------- 64 bits
def exact(case, seed):
    """From the definitions, row by row of the softmax, in 64 bits."""
    st = prepare(case, seed)
    c, k = case, case["kind"]
    f8 = torch.float64
    if k == "train_window":
        return _train64(st)
    if k == "evict":
        return _evict64(st)
    if k in ("decode_window", "decode_weighted"):
        G = c["Hq"] // c["Hkv"]
        outs, ws = [], []
        for layer in range(c["L"]):
            out = torch.zeros((c["B"], c["Hq"], c["D"]), device=DEV, dtype=f8)
            w = st["w"][layer].to(f8) if k == "decode_weighted" else None
            for b, n in enumerate(st["lens"]):
                if n == 0:
                    continue
                j = torch.arange(n, device=DEV)
                win = c.get("window", 0)
                seen = (j >= n - win) | (j < c["sinks"]) if win else torch.ones_like(j, dtype=torch.bool)
                idx = j[seen]
                K, V = _rows(st["kv"][layer], 0, st["bt"][layer][b], idx, c["page"], f8)
                x = torch.einsum("hgd,jhd->hgj", st["q"][layer][b].to(f8).view(c["Hkv"], G, c["D"]), K) / c["D"] ** 0.5
                p = torch.softmax(x, -1)
                out[b] = torch.einsum("hgj,jhd->hgd", p, V).reshape(c["Hq"], c["D"])
                if w is not None:
                    for u in range(c["units"]):
                        part = p[u] if c["units"] > 1 else p.reshape(-1, n)
                        w[b, u, :n] += part.sum(0)
            outs.append(out)
            ws.append(w)
        return outs if k == "decode_window" else (outs, ws)
    G = c["Hq"] // c["Hkv"]
    T = st["q"].shape[0]
    out = torch.zeros((T, c["Hq"], 128), device=DEV, dtype=f8)
    lse = torch.zeros((T, c["Hq"]), device=DEV, dtype=f8)
    w = st["w"].to(f8) if k == "prompt_weights" else None
    qs = st["qs"].tolist()
    for r, n in enumerate(st["lens"]):
        K, V = _rows(st["kv"], c["layout"], st["bt"][r], torch.arange(n, device=DEV), c["page"], f8)
        nq = qs[r + 1] - qs[r]
        j = torch.arange(n, device=DEV)
        for a in range(0, nq, 512):
            i = torch.arange(a, min(a + 512, nq), device=DEV)
            if w is not None and c["observe"]:
                i = i[i >= nq - c["observe"]]
                if not len(i):
                    continue
            p0 = (n - nq + i)[:, None]
            far = (p0 - j >= c["window"]) & (j >= c["sinks"]) if c["window"] else torch.zeros_like(p0 < j)
            bias = torch.zeros((len(i), n), device=DEV, dtype=f8)
            bias[(j > p0) | far] = float("-inf")
            for h in range(c["Hq"]):
                x = st["q"][qs[r] + i, h].to(f8) @ K[:, h // G].t() / 128 ** 0.5 + bias
                if w is None:
                    out[qs[r] + i, h] = torch.softmax(x, -1) @ V[:, h // G]
                    lse[qs[r] + i, h] = torch.logsumexp(x, -1)
                else:
                    w[r, h // G if c["units"] > 1 else 0, :n] += torch.exp(
                        x - st["lse"][qs[r] + i, h].to(f8)[:, None]).sum(0)
    return (out, lse) if w is None else w


def _train64(st):
    c = st["c"]
    f8 = torch.float64
    q, k, v = (st[x].detach() for x in ("q", "k", "v"))
    G = c["H"] // c["Hkv"]
    i = torch.arange(c["S"], device=DEV)
    seen = (i[None] <= i[:, None]) & ((i[:, None] - i[None] < c["window"]) | (i[None] < c["sinks"]))
    bias = torch.zeros(seen.shape, device=DEV, dtype=f8).masked_fill_(~seen, float("-inf"))
    out = torch.empty(q.shape, device=DEV, dtype=f8)
    dq, dk, dv = out.clone(), torch.zeros(k.shape, device=DEV, dtype=f8), torch.zeros(v.shape, device=DEV, dtype=f8)
    for b in range(c["B"]):
        for h in range(c["H"]):
            a = [t.to(f8).requires_grad_(True) for t in (q[b, h], k[b, h // G], v[b, h // G])]
            o = torch.softmax(a[0] @ a[1].t() / c["D"] ** 0.5 + bias, -1) @ a[2]
            gr = torch.autograd.grad(o, a, st["do"][b, h].to(f8))
            out[b, h] = o.detach()
            dq[b, h] = gr[0]
            dk[b, h // G] += gr[1]
            dv[b, h // G] += gr[2]
    return out, dq, dk, dv


def _evict64(st):
    c = st["c"]
    page = c["page"]
    kv = [x.clone() for x in st["kv"]]
    new, ws, keeps = [], [], []
    for layer in range(c["L"]):
        wt = st["w"][layer].to(torch.float64).cpu().numpy()
        W = np.zeros_like(wt)
        keep = np.full((c["B"], c["units"], c["budget"]), -1, dtype=np.int32)
        src, dst = st["bt"][layer].cpu().numpy(), st["dst"][layer].cpu().numpy()
        heads = [slice(None)] if c["units"] == 1 else [slice(u, u + 1) for u in range(c["units"])]
        for b, n in enumerate(st["lens"]):
            for u, hd in enumerate(heads):
                order = wt[b, u, :n].copy()
                order[:c["sinks"]] = np.inf
                order[n - min(n, c["recent"]):] = np.inf
                rows = np.sort(np.lexsort((np.arange(n), -order))[:c["budget"]])
                keep[b, u, :len(rows)] = rows
                W[b, u, :len(rows)] = wt[b, u, rows]
                to = np.arange(len(rows))
                t = [torch.from_numpy(x.astype(np.int64)).to(DEV)
                     for x in (src[b, rows // page], rows % page, dst[b, to // page], to % page)]
                kv[layer][:, :, :, hd][t[2], :, t[3]] = st["kv"][layer][:, :, :, hd][t[0], :, t[1]]
        new.append(torch.tensor([min(n, c["budget"]) for n in st["lens"]], dtype=torch.int32, device=DEV))
        ws.append(torch.from_numpy(W).to(DEV))
        keeps.append(torch.from_numpy(keep).to(DEV))
    return dict(kv=kv, new_lens=new, weights=ws, keep=keeps)


# ---------------------------------------------------------------- what a pass cannot do without
def _pairs(nq, n, window, sinks):
    """Visible (row, key) pairs of the last nq of n positions."""
    p = np.arange(n - nq, n, dtype=np.int64)
    if window <= 0:
        return int((p + 1).sum())
    lo = np.maximum(0, p - window + 1)
    return int((p + 1 - lo + np.minimum(sinks, lo)).sum())


def work(case):
    c, k = case, case["kind"]
    if k in ("decode_window", "decode_weighted"):
        rows = 0
        for n in _lens(c):
            s, w = _visible_span(n, c.get("window", 0), c.get("sinks", 0))
            rows += n - w + s
        by = c["L"] * (rows * c["Hkv"] * c["D"] * 4 + 2 * c["B"] * c["Hq"] * c["D"] * 2)
        if k == "decode_weighted":
            by += c["L"] * rows * c["units"] * 8
        return dict(bytes=by, flops=c["L"] * 4 * c["Hq"] * rows * c["D"])
    if k in ("prompt_window", "prompt_weights"):
        q, lens = _lens(c)
        obs = c.get("observe", 0)
        used = [min(x, obs) if obs else x for x in q]
        pairs = sum(_pairs(a, n, c["window"], c["sinks"]) for a, n in zip(used, lens))
        rows = 0
        for a, n in zip(used, lens):
            s, w = _visible_span(n - a + 1, c["window"], c["sinks"])
            rows += n - w + s
        kv, tok = rows * c["Hkv"] * 256, sum(used) * c["Hq"]
        if k == "prompt_window":
            return dict(bytes=2 * kv + tok * (512 + 4), flops=4 * 128 * pairs * c["Hq"])
        return dict(bytes=kv + tok * (256 + 4) + rows * c["units"] * 8, flops=2 * 128 * pairs * c["Hq"])
    if k == "train_window":
        pairs = _pairs(c["S"], c["S"], c["window"], c["sinks"]) * c["B"] * c["H"]
        x = c["B"] * c["S"] * c["D"] * 2
        # forward and backward: q, k, v, dO in; out, dq, dk, dv out
        return dict(bytes=x * (4 * c["H"] + 4 * c["Hkv"]), flops=14 * c["D"] * pairs)
    kept = sum(min(n, c["budget"]) for n in _lens(c))
    n = sum(_lens(c))
    cap = c["B"] * ((max(c["hi"], 1) + c["page"] - 1) // c["page"] * c["page"])
    return dict(bytes=c["L"] * (kept * c["Hkv"] * c["D"] * 8 + c["units"] * 4 * (n + cap + c["B"] * c["budget"])),
                flops=c["L"] * c["units"] * n)
