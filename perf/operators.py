"""What is measured of the operators for speculative decoding over a tree of drafted tokens.

Four operators, each in a plain form (elementary torch operations in 32 bits,
rounded once at the end) and as the call a user makes of ``myinfer_b200.tree``:

* ``attention``  ``tree_attention``: every node of a drafted tree attends to its
                 sequence's cache and to its ancestors in the tree;
* ``logits``     ``process_logits``: penalties for repeated tokens (the
                 sequence's counts plus the tokens on the node's own path), biases
                 and a grammar's bit mask on the logits, and the greedy choice;
* ``accept``     ``tree_accept``: the longest path of drafted tokens that equal the
                 model's own choices, and the counts that follow from it;
* ``commit``     ``commit_tree``: the accepted rows of every layer's cache moved
                 behind the prefix.

``own`` selects the framework's calls.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEV = "cuda"


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one new token of a short chat on the smallest dense shape: latency only
        dict(name="attention_one_512", op="attention", batch=1, heads=16, kv_heads=8, dim=128, rows=1, tree=1,
             keys=512, bits=8),
        # four requests of different lengths, 13 drafted tokens each, over 4-bit caches (the 32/4-head MoE shape)
        dict(name="attention_batch_4k", op="attention", batch=4, heads=32, kv_heads=4, dim=128, rows=13, tree=13,
             keys=4111, bits=4),
        # the last level of a 31-node tree (16 rows) over an unquantized cache of small heads, before quantization starts
        dict(name="attention_bf16_2500", op="attention", batch=2, heads=8, kv_heads=2, dim=64, rows=16, tree=31,
             keys=2500, bits=0),
        # a full tree of 64 nodes at the dense benchmark's context: the largest arithmetic
        dict(name="attention_64_32k", op="attention", batch=1, heads=64, kv_heads=8, dim=128, rows=64, tree=64,
             keys=32768, bits=8),
        # 16 drafted tokens at the longest context of the attention benchmark: the largest cache
        dict(name="attention_16_128k", op="attention", batch=1, heads=64, kv_heads=8, dim=128, rows=16, tree=16,
             keys=131072, bits=4),
        # one row of plain decoding with penalties only
        dict(name="logits_one", op="logits", batch=1, tree=1, vocab=151936, dtype="bf16", penalties=True, bias=0,
             mask=False),
        # a whole tree's rows with everything on: the step a constrained request pays for each verification
        dict(name="logits_tree_64", op="logits", batch=1, tree=64, vocab=151936, dtype="bf16", penalties=True,
             bias=300, mask=True),
        # a batch of small trees, 32-bit logits of a vocabulary that is no multiple of a vector
        dict(name="logits_batch_odd", op="logits", batch=8, tree=5, vocab=32001, dtype="f32", penalties=True,
             bias=17, mask=True),
        # one request's small tree
        dict(name="accept_one", op="accept", batch=1, tree=8, vocab=151936),
        # a full batch of full trees
        dict(name="accept_batch", op="accept", batch=64, tree=64, vocab=151936),
        # a small dense model's cache after a short tree
        dict(name="commit_28_layers", op="commit", layers=28, batch=1, kv_heads=8, dim=128, tree=15, keys=1024, bits=8),
        # the largest dense shape's depth, four requests
        dict(name="commit_64_layers", op="commit", layers=64, batch=4, kv_heads=8, dim=128, tree=64, keys=700, bits=4),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "logits", "logits", "accept", "commit"])
    if op == "attention":
        kv = rng.choice([1, 2, 4, 8])
        group = rng.choice([1, 2, 4, 5, 8, 16])
        dim = rng.choice([64, 128, 128])
        bits = rng.choice([0, 4, 8])
        tree = rng.choice([1, _log(rng, 2, 64)])
        rows = rng.choice([tree, max(1, tree - rng.randrange(tree))])
        batch = rng.choice([1, 1, _log(rng, 2, 16)])
        most = min(131072, (8 * 131072) // (kv * batch), (64 * 64 * 32768) // (batch * kv * group * rows))
        return dict(op=op, batch=batch, heads=kv * group, kv_heads=kv, dim=dim, rows=rows, tree=tree,
                    keys=_log(rng, 1, most), bits=bits)
    if op == "logits":
        tree = rng.choice([1, _log(rng, 2, 64)])
        batch = max(1, min(_log(rng, 1, 64), 64 // tree))
        vocab = rng.choice([151936, _log(rng, 1000, 151936)])
        return dict(op=op, batch=batch, tree=tree, vocab=vocab, dtype=rng.choice(["bf16", "bf16", "f32"]),
                    penalties=rng.random() < 0.8, bias=rng.choice([0, _log(rng, 1, 300)]), mask=rng.random() < 0.6)
    if op == "accept":
        return dict(op=op, batch=_log(rng, 1, 64), tree=_log(rng, 1, 64), vocab=_log(rng, 1000, 151936))
    return dict(op=op, layers=_log(rng, 2, 64), batch=_log(rng, 1, 4), kv_heads=rng.choice([1, 2, 4, 8]),
                dim=rng.choice([64, 128]), tree=_log(rng, 1, 64), keys=_log(rng, 1, 1024), bits=rng.choice([0, 4, 8]))


def _lengths(case):
    """Prefix lengths of the requests of a batch: the longest first, the last one 30 % of it."""
    B, n = case["batch"], case["keys"]
    return [int(n * (1.0 - 0.7 * b / max(1, B - 1))) if B > 1 else n for b in range(B)]


# ------------------------------------------------------------------ inputs
def _rng(seed):
    return np.random.default_rng(int(seed))


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) * 7919 + 13)
    return g


def _parents(rng, B, T):
    """Random drafted trees in level-like order: parents[0] = -1, 0 <= parents[i] < i after it."""
    p = np.full((B, T), -1, np.int32)
    for i in range(1, T):
        p[:, i] = np.maximum(0, i - 1 - rng.integers(0, np.minimum(i, 9), B))
    return p


def _ancestors(parents):
    """int64 [B, T]: bit j of row i is set where j is i or an ancestor of i."""
    B, T = parents.shape
    bits = np.zeros((B, T), np.uint64)
    for i in range(T):
        own_bit = np.uint64(1) << np.uint64(i)
        up = bits[np.arange(B), np.maximum(parents[:, i], 0)] if i else np.zeros(B, np.uint64)
        bits[:, i] = up | own_bit
    return bits.view(np.int64)


def _packed(x, bits):
    """Affine groups of 64 along the last axis: (packed int32 words, bf16 scales, bf16 biases)."""
    lead, D = x.shape[:-1], x.shape[-1]
    g = x.reshape(*lead, D // 64, 64)
    lo, hi = g.amin(-1), g.amax(-1)
    s = ((hi - lo) / (2 ** bits - 1)).clamp_min(1e-6).to(torch.bfloat16)
    b = lo.to(torch.bfloat16)
    c = ((g - b.float()[..., None]) / s.float()[..., None]).round_().clamp_(0, 2 ** bits - 1).to(torch.int32)
    c = c.reshape(*lead, D * bits // 32, 32 // bits)
    w = torch.zeros(c.shape[:-1], dtype=torch.int32, device=x.device)
    for i in range(32 // bits):
        w |= c[..., i] << (bits * i)
    return w, s, b


def _kv(g, shape, bits, outliers):
    x = torch.randn(shape, generator=g, device=DEV)
    if outliers:  # keys have a few channels of much larger size
        x[..., ::37] *= 4.0
    return _packed(x, bits) if bits else x.to(torch.bfloat16)


def prepare(case, seed):
    rng, g, op = _rng(seed), _gen(seed), case["op"]
    s = dict(case=case)
    if op == "attention":
        B, Hq, Hk, D, L, T = (case[k] for k in ("batch", "heads", "kv_heads", "dim", "rows", "tree"))
        cap = (case["keys"] + T + 255) // 256 * 256
        s["q"] = (1.5 * torch.randn(B, Hq, L, D, generator=g, device=DEV)).to(torch.bfloat16)
        s["k"] = _kv(g, (B, Hk, cap, D), case["bits"], True)
        s["v"] = _kv(g, (B, Hk, cap, D), case["bits"], False)
        anc = _ancestors(_parents(rng, B, T))[:, T - L:]  # the tree's last L nodes ask
        s["ancestors"] = torch.from_numpy(anc.copy()).to(DEV)
        s["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device=DEV)
    elif op == "logits":
        B, T, V = case["batch"], case["tree"], case["vocab"]
        R = B * T
        x = 2.5 * torch.randn(R, V, generator=g, device=DEV)
        top = torch.randint(0, V, (R, 40), generator=g, device=DEV)
        x.scatter_add_(1, top, 10 * torch.rand(R, 40, generator=g, device=DEV))
        s["logits"] = x.to(torch.bfloat16 if case["dtype"] == "bf16" else torch.float32)
        s["counts"] = s["penalties"] = s["tokens"] = s["ancestors"] = None
        s["bias_ids"] = s["bias_values"] = s["mask"] = None
        if case["penalties"]:
            counts = torch.zeros(B, V, dtype=torch.int32, device=DEV)
            seen = torch.randint(0, V, (B, 2000), generator=g, device=DEV)
            counts.scatter_add_(1, seen, torch.ones_like(seen, dtype=torch.int32))
            counts.scatter_add_(1, top.reshape(B, -1)[:, :30].contiguous(),
                                torch.ones(B, 30, dtype=torch.int32, device=DEV))
            s["counts"] = counts
            pen = np.stack([1.05 + 0.3 * rng.random(B), rng.random(B), 0.5 * rng.random(B)], 1)
            s["penalties"] = torch.from_numpy(pen.astype(np.float32)).to(DEV)
            if T > 1:
                tok = top.reshape(B, T, 40)[:, :, 0].to(torch.int32)
                s["tokens"] = tok.contiguous()
                s["ancestors"] = torch.from_numpy(_ancestors(_parents(rng, B, T))).to(DEV)
        if case["bias"]:
            ids = np.stack([rng.choice(V, case["bias"], replace=False) for _ in range(B)]).astype(np.int32)
            s["bias_ids"] = torch.from_numpy(ids).to(DEV)
            s["bias_values"] = 4 * torch.randn(B, case["bias"], generator=g, device=DEV)
        if case["mask"]:
            # what grammars leave of a vocabulary: a handful of tokens, a class of them, or nearly all
            share = torch.from_numpy(rng.choice([0.0005, 0.3, 0.98], R)).to(DEV)
            if R >= 16:
                share[-1] = -1.0  # a dead end leaves nothing
            W = (V + 31) // 32
            m = torch.zeros(R, W, dtype=torch.int32, device=DEV)
            for i in range(32):
                m |= (torch.rand(R, W, generator=g, device=DEV) < share[:, None]).to(torch.int32) << i
            s["mask"] = m
    elif op == "accept":
        B, T, V = case["batch"], case["tree"], case["vocab"]
        par = _parents(rng, B, T)
        tok = rng.integers(0, V, (B, T)).astype(np.int32)
        pick = rng.integers(0, V, (B, T)).astype(np.int32)
        for b in range(B):  # most nodes have a child that the model agrees with
            for i in range(1, T):
                if rng.random() < 0.7:
                    pick[b, par[b, i]] = tok[b, i]
        s["parents"], s["tokens"], s["picks"] = (torch.from_numpy(a).to(DEV) for a in (par, tok, pick))
        s["counts"] = torch.zeros(B, V, dtype=torch.int32, device=DEV)
    else:
        NL, B, Hk, D, T, bits = (case[k] for k in ("layers", "batch", "kv_heads", "dim", "tree", "bits"))
        cap = (case["keys"] + T + 255) // 256 * 256
        if bits:
            W = D * bits // 32
            parts = [torch.randint(-2 ** 31, 2 ** 31 - 1, (NL, B, Hk, cap, W), generator=g, device=DEV,
                                   dtype=torch.int32) for _ in range(2)]
            small = [torch.randn(NL, B, Hk, cap, D // 64, generator=g, device=DEV).to(torch.bfloat16)
                     for _ in range(4)]
            s["buffers"] = [parts[0], small[0], small[1], parts[1], small[2], small[3]]
            s["layers"] = [(tuple(t[i] for t in s["buffers"][:3]), tuple(t[i] for t in s["buffers"][3:]))
                           for i in range(NL)]
        else:
            s["buffers"] = [torch.randn(NL, B, Hk, cap, D, generator=g, device=DEV).to(torch.bfloat16)
                            for _ in range(2)]
            s["layers"] = [(s["buffers"][0][i], s["buffers"][1][i]) for i in range(NL)]
        par = _parents(rng, B, T)
        path = np.full((B, T), -1, np.int32)
        n = np.zeros(B, np.int32)
        for b in range(B):  # the path from a random deep node up to the root
            node, up = int(rng.integers(T // 2, T)), []
            while node >= 0:
                up.append(node)
                node = int(par[b, node])
            n[b] = len(up)
            path[b, :len(up)] = up[::-1]
        s["path"], s["accepted"] = torch.from_numpy(path).to(DEV), torch.from_numpy(n).to(DEV)
        s["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device=DEV)
    return s


# ------------------------------------------------------------------ plain forms
def _codes(w, bits):
    sh = torch.arange(0, 32, bits, device=w.device, dtype=torch.int32)
    return ((w[..., None] >> sh) & (2 ** bits - 1)).reshape(*w.shape[:-1], -1)


def _dense(t, bits):
    if not bits:
        return t.float()
    w, s, b = t
    c = _codes(w, bits).float()
    c = c.reshape(*c.shape[:-1], -1, 64)
    return (c * s.float()[..., None] + b.float()[..., None]).flatten(-2)


def _plain_attention(s):
    c, q = s["case"], s["q"].float()
    B, Hq, L, D = q.shape
    k, v = _dense(s["k"], c["bits"]), _dense(s["v"], c["bits"])
    Hk, S = k.shape[1], k.shape[2]
    T = c["tree"]
    key = torch.arange(S, device=q.device)
    node = key[None] - s["lengths"][:, None]                       # [B, S] tree index of each key
    bit = (s["ancestors"][:, :, None] >> node.clamp(0, 63)[:, None]) & 1
    see = (node < 0)[:, None] | ((node >= 0) & (node < T))[:, None] & (bit == 1)  # [B, L, S]
    x = torch.matmul(q.reshape(B, Hk, -1, D) * D ** -0.5, k.transpose(-1, -2)).reshape(B, Hk, Hq // Hk, L, S)
    x = x.masked_fill(~see[:, None, None], -math.inf)
    m = x.amax(-1, keepdim=True).clamp_min(-3e38)
    p = torch.exp(x - m)
    den = p.sum(-1)
    v = v * see.any(1)[:, None, :, None]
    o = torch.matmul(p.reshape(B, Hk, -1, S), v).reshape(B, Hk, Hq // Hk, L, D)
    o = o / den.clamp_min(1e-30)[..., None]
    return o.reshape(B, Hq, L, D).to(torch.bfloat16)


def _plain_logits(s):
    x = s["logits"]
    R, V = x.shape
    B, T = s["case"]["batch"], s["case"]["tree"]
    v = x.float().reshape(B, T, V)
    if s["counts"] is not None:
        n = s["counts"][:, None].expand(B, T, V)
        if s["tokens"] is not None:
            bit = (s["ancestors"][:, :, None] >> torch.arange(T, device=x.device)) & 1  # [B, T, T]
            idx = s["tokens"].long()[:, None].expand(B, T, T)
            n = n.contiguous().scatter_add_(2, idx, bit.to(torch.int32))
        rep, pres, freq = (s["penalties"][:, i, None, None] for i in range(3))
        seen = n > 0
        v = torch.where(seen, torch.where(v < 0, v * rep, v / rep), v)
        v = torch.where(seen, v - pres, v)
        v = torch.where(seen, v - freq * n.float(), v)
    if s["bias_ids"] is not None:
        d = torch.zeros(B, V, device=x.device).scatter_(1, s["bias_ids"].long(), s["bias_values"])
        v = v + d[:, None]
    if s["mask"] is not None:
        ok = ((s["mask"][..., None] >> torch.arange(32, device=x.device, dtype=torch.int32)) & 1).reshape(R, -1)
        v = torch.where(ok[:, :V].reshape(B, T, V) == 1, v, -math.inf)
    out = v.reshape(R, V).to(x.dtype)
    f = torch.where(torch.isnan(out), -math.inf, out.float())
    top = f.amax(-1, keepdim=True)
    at = torch.where(f == top, torch.arange(V, device=x.device), V).amin(-1)
    return out, torch.where(top[:, 0] == -math.inf, -1, at).to(torch.int32)


def _plain_accept(s):
    par, tok, pick = s["parents"].long(), s["tokens"], s["picks"]
    B, T = par.shape
    i = torch.arange(T, device=par.device)
    hit = (torch.gather(pick, 1, par.clamp_min(0)) == tok) & (par >= 0)
    # the first of the siblings that match
    twin = (par[:, :, None] == par[:, None, :]) & hit[:, None, :] & (i[None] < i[:, None])
    hit = hit & ~twin.any(2)
    hit[:, 0] = True
    # accepted: the node and all its ancestors match (reach[i, j]: j is i or above it, by squaring)
    reach = (torch.nn.functional.one_hot(par.clamp_min(0), T) * (par >= 0)[..., None]).float() + torch.eye(T, device=par.device)
    for _ in range(max(1, (T - 1).bit_length())):
        reach = (torch.matmul(reach, reach) > 0).float()
    good = torch.matmul(reach, (~hit).float()[..., None])[..., 0] == 0
    n = good.sum(1).to(torch.int32)
    path = torch.where(good, i, T).sort(1).values
    last = torch.gather(path, 1, (n.long() - 1)[:, None])
    nxt = torch.gather(pick, 1, last)[:, 0]
    s["counts"].scatter_add_(1, tok.long(), good.to(torch.int32))
    return torch.where(path < T, path, -1).to(torch.int32), n, nxt, s["counts"]


def _plain_commit(s):
    n = s["accepted"]
    B, T = s["path"].shape
    base = s["lengths"].long()
    i = torch.arange(T, device=base.device)
    live = i[None] < n[:, None]
    src = torch.where(live, base[:, None] + s["path"], base[:, None] + i)
    dst = base[:, None] + i
    b = torch.arange(B, device=base.device)[:, None]
    for t in s["buffers"]:
        t[:, b, :, dst] = t[:, b, :, src]
    return [t.view(torch.int16) if t.dtype == torch.bfloat16 else t for t in s["buffers"]]


def run(state):
    op = state["case"]["op"]
    if not own:
        return dict(attention=_plain_attention, logits=_plain_logits, accept=_plain_accept,
                    commit=_plain_commit)[op](state)
    from myinfer_b200 import tree
    c = state["case"]
    if op == "attention":
        return tree.tree_attention(state["q"], state["k"], state["v"], state["lengths"], state["ancestors"],
                                   c["dim"] ** -0.5, tree_len=c["tree"], bits=c["bits"])
    if op == "logits":
        return tree.process_logits(state["logits"], batch=c["batch"], counts=state["counts"],
                                   penalties=state["penalties"], tokens=state["tokens"],
                                   ancestors=state["ancestors"], bias_ids=state["bias_ids"],
                                   bias_values=state["bias_values"], mask=state["mask"])
    if op == "accept":
        path, n, nxt = tree.tree_accept(state["parents"], state["tokens"], state["picks"], counts=state["counts"])
        return path, n, nxt, state["counts"]
    # a decoding loop keeps the table of its cache's buffers until they are reallocated
    table = state.get("table") or state.setdefault("table", tree.CacheLayers(state["layers"]))
    tree.commit_tree(table, state["lengths"], state["path"], state["accepted"])
    return [t.view(torch.int16) if t.dtype == torch.bfloat16 else t for t in state["buffers"]]


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    op = case["op"]
    if op == "attention":
        B, Hq, Hk, D, L, T = (case[k] for k in ("batch", "heads", "kv_heads", "dim", "rows", "tree"))
        row = D * case["bits"] // 8 + D // 64 * 4 if case["bits"] else 2 * D
        keys = sum(_lengths(case)) + B * T
        return dict(bytes=2 * Hk * row * keys + 4 * B * Hq * L * D + 8 * B * L, flops=4 * Hq * L * D * keys)
    if op == "logits":
        B, T, V = case["batch"], case["tree"], case["vocab"]
        size = 2 if case["dtype"] == "bf16" else 4
        n = 2 * size * B * T * V + 4 * B * T
        n += 4 * B * V if case["penalties"] else 0
        n += 8 * B * case["bias"] + (B * T * ((V + 31) // 32) * 4 if case["mask"] else 0)
        return dict(bytes=n, flops=B * T * V * (1 + 4 * case["penalties"]))
    if op == "accept":
        B, T = case["batch"], case["tree"]
        return dict(bytes=16 * B * T + 8 * B, flops=4 * B * T)
    NL, B, Hk, D, T = (case[k] for k in ("layers", "batch", "kv_heads", "dim", "tree"))
    row = D * case["bits"] // 8 + D // 64 * 4 if case["bits"] else 2 * D
    rows = max(1, round(0.3 * T))  # about what a random path of these trees moves
    return dict(bytes=2 * 2 * NL * B * Hk * row * rows, flops=0)


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    if case["op"] in ("accept", "commit"):
        return None  # whole numbers and moved bits
    s = prepare(case, seed)
    if case["op"] == "attention":
        return _exact_attention(case, s)
    R, V = s["logits"].shape
    T = case["tree"]
    out = np.empty((R, V))
    x = s["logits"].double().cpu().numpy()
    host = {k: (None if s[k] is None else s[k].cpu().numpy()) for k in
            ("counts", "penalties", "tokens", "ancestors", "bias_ids", "bias_values", "mask")}
    for r in range(R):
        b, t = divmod(r, T)
        y = x[r].copy()
        if host["counts"] is not None:
            n = host["counts"][b].astype(np.int64).copy()
            if host["tokens"] is not None:
                a = int(host["ancestors"][b, t])
                for j in range(T):
                    if a >> j & 1:
                        n[host["tokens"][b, j]] += 1
            rep, pres, freq = (float(z) for z in host["penalties"][b])
            at = np.nonzero(n)[0]
            z = y[at]
            y[at] = np.where(z < 0, z * rep, z / rep) - pres - freq * n[at]
        if host["bias_ids"] is not None:
            y[host["bias_ids"][b]] += host["bias_values"][b].astype(np.float64)
        if host["mask"] is not None:
            ok = np.unpackbits(host["mask"][r].view(np.uint8), bitorder="little")[:V]
            y[ok == 0] = -np.inf
        out[r] = y
    return torch.from_numpy(out), None


def _exact_attention(case, s):
    B, Hq, Hk, D, L, T = (case[k] for k in ("batch", "heads", "kv_heads", "dim", "rows", "tree"))
    bits, G = case["bits"], Hq // Hk
    lens = _lengths(case)
    anc = s["ancestors"].cpu().numpy().view(np.uint64)
    out = torch.zeros(B, Hq, L, D, dtype=torch.float64)

    def head(t, b, h, n):
        if not bits:
            return t[b, h, :n].double()
        w, sc, bi = (u[b, h, :n] for u in t)
        per = 32 // bits
        x = torch.empty(n, D, dtype=torch.float64, device=w.device)
        for i in range(per):
            x[:, i::per] = torch.bitwise_and(torch.bitwise_right_shift(w, bits * i), 2 ** bits - 1).double()
        return x * sc.double().repeat_interleave(64, 1) + bi.double().repeat_interleave(64, 1)

    for b in range(B):
        n = lens[b]
        hide = torch.zeros(L, n + T, dtype=torch.float64)
        for i in range(L):
            for j in range(T):
                if not int(anc[b, i]) >> j & 1:
                    hide[i, n + j] = -math.inf
        hide = hide.to(s["q"].device)
        for h in range(Hk):
            k, v = head(s["k"], b, h, n + T), head(s["v"], b, h, n + T)
            for g in range(G):
                z = s["q"][b, h * G + g].double() @ k.T / math.sqrt(D) + hide
                w = torch.exp(z - torch.logsumexp(z, 1, keepdim=True))
                out[b, h * G + g] = (w @ v).cpu()
    return out
