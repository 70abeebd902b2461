"""The tree-speculation operators (myinfer_b200.tree) against their definitions in 64 bits.

Attention's tolerance, per output element, from the roundings the kernel may
make (u = 2^-11, fp16's unit roundoff): a key element that is used in fp16 is
off by at most u times its value, and the D independent errors of a score add
up like their root sum of squares; 8 / sqrt(3) of it is no less than 8 standard
deviations.  A score off by d changes every weight by a factor in exp(+-2d).  Weights and values in
fp16 add 2 u, fp32 sums less than u more.  The output's rounding to bf16 is half a unit, at most
2^-8 of the value.  So
  |d| <= 2^-8 |ref| + (2 d + 4 u) sum(p |v|)
and in the 2-norm, over everything, 5e-3 (bf16 rounding alone is 1.7e-3)."""

import math

import numpy as np
import pytest
import torch

from oracle import tree as ref

pytestmark = pytest.mark.gpu
U = 2.0 ** -11


def _bf(x):
    return torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32)).to(torch.bfloat16)


def _f64(t):
    return t.double().cpu().numpy()


def _pack(x, bits):
    """numpy fp32 [..., D] -> MLX tuple of torch CPU tensors."""
    g = x.reshape(*x.shape[:-1], -1, 64)
    lo, hi = g.min(-1), g.max(-1)
    s, b = _bf((hi - lo) / (2 ** bits - 1)), _bf(lo)
    sf, bfv = s.float().numpy(), b.float().numpy()
    with np.errstate(divide="ignore", invalid="ignore"):
        c = np.nan_to_num((g - bfv[..., None]) / sf[..., None])
    c = np.clip(np.rint(c), 0, 2 ** bits - 1).astype(np.uint32).reshape(*x.shape[:-1], -1, 32 // bits)
    w = np.zeros(c.shape[:-1], np.uint32)
    for i in range(32 // bits):
        w |= c[..., i] << np.uint32(bits * i)
    return torch.from_numpy(w.view(np.int32)), s, b


def _cache(rng, B, H, rows, D, bits, size=1.0):
    x = (size * rng.standard_normal((B, H, rows, D))).astype(np.float32)
    return _pack(x, bits) if bits else _bf(x)


def _dense(t, bits):
    """fp64 values of a CPU cache."""
    return ref.dequant((t[0].numpy(), _f64(t[1]), _f64(t[2])), bits) if bits else _f64(t)


def _cuda(t):
    return tuple(x.cuda() for x in t) if isinstance(t, tuple) else t.cuda()


def _trees(rng, B, T):
    p = np.full((B, T), -1, np.int32)
    for i in range(1, T):
        p[:, i] = rng.integers(max(0, i - 5), i, B)
    return p


def _attend(q, k, v, lengths, words, scale, T, bits, **kw):
    from myinfer_b200.tree import tree_attention
    return tree_attention(q, _cuda(k), _cuda(v), torch.tensor(lengths, dtype=torch.int32).cuda(),
                          torch.from_numpy(words.view(np.int64).copy()).cuda(), scale, tree_len=T, bits=bits, **kw)


def _check(out, q, k, v, lengths, words, scale, T, bits):
    out, q = _f64(out), _f64(q)
    kd, vd = _dense(k, bits), _dense(v, bits)
    B, Hq, L, D = q.shape
    Hk = kd.shape[1]
    num = den = 0.0
    for b in range(B):
        end = min(lengths[b] + T, kd.shape[2])
        kb, vb = (np.nan_to_num(x[b, :, :end], nan=0, posinf=0, neginf=0) for x in (kd, vd))
        want, mag = ref.attention(q[b], kb, vb, lengths[b], words[b], T, scale)
        tol = 2.0 ** -8 * np.abs(want) + 1e-30
        for h in range(Hq):
            hk = h // (Hq // Hk)
            if end:
                d = 8 / math.sqrt(3) * U * abs(scale) * np.sqrt((q[b, h] ** 2) @ (kb[hk] ** 2).T).max(1)
                tol[h] += (np.expm1(np.minimum(2 * d, 1.0)) + 4 * U)[:, None] * mag[h]
        assert np.isfinite(out[b]).all()
        err = np.abs(out[b] - want)
        assert (err <= tol).all(), (b, float((err - tol).max()), np.argwhere(err > tol)[:4])
        num, den = num + (err ** 2).sum(), den + (want ** 2).sum()
    if den:
        assert math.sqrt(num / den) <= 5e-3, math.sqrt(num / den)


GRID = [  # B, Hq, Hkv, L, T, lengths, spare rows
    (1, 8, 8, 1, 1, [0], 3),            # the first token of an empty cache
    (1, 2, 1, 1, 1, [1], 0),            # a cache that ends with the tree
    (1, 16, 8, 1, 1, [63], 9),
    (1, 64, 8, 1, 1, [1500], 0),
    (3, 4, 4, 1, 1, [0, 64, 129], 1),   # plain decoding of different lengths
    (2, 10, 2, 7, 7, [1, 700], 5),      # a group of five heads
    (1, 32, 2, 5, 5, [513], 2),         # a group of sixteen
    (1, 8, 2, 17, 17, [100], 0),        # 68 rows per kv head
    (4, 8, 4, 13, 13, [0, 3, 250, 1023], 7),
    (1, 64, 8, 64, 64, [333], 1),       # 512 rows per kv head
    (1, 16, 1, 64, 64, [2100], 30),     # 1024 rows on one kv head
    (2, 4, 2, 16, 31, [65, 31], 4),     # the newest 16 of 31 nodes
    (1, 6, 3, 1, 64, [200], 0),
    (17, 2, 1, 3, 3, [11 * i for i in range(17)], 6),
]


@pytest.mark.parametrize("bits", [0, 4, 8])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("shape", GRID, ids=lambda s: "b%d_h%dx%d_l%d_t%d_n%d" % (*s[:5], max(s[5])))
def test_attention(shape, D, bits):
    B, Hq, Hk, L, T, lengths, spare = shape
    rng = np.random.default_rng(sum(lengths) + 7 * D + bits)
    rows = max(lengths) + T + spare
    q = _bf(1.5 * rng.standard_normal((B, Hq, L, D))).cuda()
    k, v = _cache(rng, B, Hk, rows, D, bits), _cache(rng, B, Hk, rows, D, bits)
    words = ref.ancestors(_trees(rng, B, T))[0][:, T - L:]
    out = _attend(q, k, v, lengths, words, D ** -0.5, T, bits)
    _check(out, q, k, v, lengths, words, D ** -0.5, T, bits)
    again = _attend(q, k, v, lengths, words, D ** -0.5, T, bits)
    assert torch.equal(out, again)  # no order of CTAs changes a result


@pytest.mark.parametrize("bits", [0, 4, 8])
@pytest.mark.parametrize("B,Hq,Hk,L,D,n", [(1, 16, 2, 2, 128, 70001), (1, 8, 2, 64, 128, 40000), (2, 4, 2, 24, 64, 60000),
                                           (3, 24, 3, 40, 64, 9999)])
def test_attention_long(bits, B, Hq, Hk, L, D, n):
    """Dozens of tiles per CTA, so that every ring and buffer wraps many times and the warps of a CTA drift
    apart: both against the definition and from call to call.  (rel is the bound of _check's 2-norm.)"""
    from myinfer_b200 import _lib, ops
    rng = np.random.default_rng(n + bits)
    g = torch.Generator(device="cuda").manual_seed(n + bits)
    rows, lengths = n + L + 1, [n - 17 * b for b in range(B)]
    q = (1.5 * torch.randn(B, Hq, L, D, generator=g, device="cuda")).to(torch.bfloat16)
    x, y = (torch.randn(B, Hk, rows, D, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    k, v = ((ops.quantize(x, 64, bits), ops.quantize(y, 64, bits)) if bits else (x, y))
    kd, vd = ((_dense(tuple(z.cpu() for z in t), bits) for t in (k, v)) if bits else (_f64(x), _f64(y)))
    words = ref.ancestors(_trees(rng, B, L))[0]
    out = _attend(q, k, v, lengths, words, D ** -0.5, L, bits)
    for b in range(B):
        hide = np.zeros((L, lengths[b] + L))
        hide[:, lengths[b]:] = [[0.0 if int(words[b, i]) >> j & 1 else -math.inf for j in range(L)] for i in range(L)]
        hide = torch.from_numpy(hide).cuda()
        for h in range(Hq):
            kh, vh = (torch.from_numpy(t[b, h // (Hq // Hk), :lengths[b] + L]).cuda() for t in (kd, vd))
            want = torch.softmax(q[b, h].double() @ kh.T * D ** -0.5 + hide, 1) @ vh
            assert ((out[b, h].double() - want).norm() / want.norm()).item() <= 5e-3
    for _ in range(20):
        assert torch.equal(out, _attend(q, k, v, lengths, words, D ** -0.5, L, bits))
    _lib.device_check()


@pytest.mark.parametrize("bits", [0, 4, 8])
@pytest.mark.parametrize("rows", [1, 31, 33, 97, 127, 129, 161, 255])
def test_attention_rows_of_part_of_a_warp(rows, bits):
    """A warp's lanes with and without a row load tensor memory together: every count of rows around a warp's 32 and a
    block's 128, in runs that one CTA ends (few keys) and that are cut into parts."""
    rng = np.random.default_rng(rows)
    G = next(g for g in range(1, rows + 1) if rows % g == 0 and rows // g <= 64)  # heads on the one kv head
    L, D = rows // G, 128
    words = np.full((1, L), ~np.uint64(0))
    for n in (0, 1000):
        q = _bf(rng.standard_normal((1, G, L, D))).cuda()
        k, v = _cache(rng, 1, 1, n + L, D, bits), _cache(rng, 1, 1, n + L, D, bits)
        _check(_attend(q, k, v, [n], words, D ** -0.5, L, bits), q, k, v, [n], words, D ** -0.5, L, bits)


@pytest.mark.parametrize("bits", [0, 4, 8])
def test_attention_masks_and_garbage(bits):
    """Rows that see nothing are zero; rows nobody sees may hold NaN and infinities."""
    rng = np.random.default_rng(5)
    B, Hq, Hk, L, T, D = 2, 6, 2, 9, 9, 128
    lengths, rows = [0, 130], 150
    q = _bf(rng.standard_normal((B, Hq, L, D))).cuda()
    k, v = _cache(rng, B, Hk, rows, D, bits), _cache(rng, B, Hk, rows, D, bits)
    words = ref.ancestors(_trees(rng, B, T))[0]
    dead = 4  # a node no one sees, and a query that sees nothing
    words &= ~np.uint64(1 << dead)
    words[:, 2] = 0
    for t in (k, v):
        for x in (t[1:] if bits else [t]):
            for b in range(B):
                x[b, :, lengths[b] + dead] = math.nan
                x[b, :, lengths[b] + T:] = math.inf
                x[b, 0, lengths[b] + T:] = math.nan
    out = _attend(q, k, v, lengths, words, D ** -0.5, T, bits)
    assert (out[0, :, 2] == 0).all() and (out[1, :, 2] != 0).any()
    _check(out, q, k, v, lengths, words, D ** -0.5, T, bits)
    high = words | np.uint64(0xFFFF) << np.uint64(T)  # bits beyond the tree are no keys
    assert torch.equal(out, _attend(q, k, v, lengths, high, D ** -0.5, T, bits))


@pytest.mark.parametrize("bits", [0, 4, 8])
@pytest.mark.parametrize("ksize,vsize,scale", [(3e4, 1.0, 3e-6), (1e-6, 1e-6, 8e4), (1.0, 3e5, 0.09), (1.0, 1.0, -0.09),
                                               (40.0, 1.0, 0.09)])
def test_attention_ranges(bits, ksize, vsize, scale):
    """Keys and values far from 1, a negative scale, and scores of several hundred."""
    rng = np.random.default_rng(11)
    B, Hq, Hk, L, T, D = 1, 4, 2, 6, 6, 128
    lengths = [391]
    q = _bf(rng.standard_normal((B, Hq, L, D))).cuda()
    k, v = _cache(rng, B, Hk, 400, D, bits, ksize), _cache(rng, B, Hk, 400, D, bits, vsize)
    words = ref.ancestors(_trees(rng, B, T))[0]
    _check(_attend(q, k, v, lengths, words, scale, T, bits), q, k, v, lengths, words, scale, T, bits)


@pytest.mark.parametrize("bits", [0, 4, 8])
def test_attention_growing_scores(bits):
    """The running maximum moves at every tile, by more and less than the kernel may defer; values grow by 2^12 along the cache."""
    rng = np.random.default_rng(12)
    L = T = 3
    n, D = 900, 64
    grow = np.linspace(0.1, 9.0, n + T)[None, None, :, None]
    q = _bf(np.abs(rng.standard_normal((1, 2, L, D)))).cuda()
    kx = (np.abs(rng.standard_normal((1, 1, n + T, D))) * grow).astype(np.float32)
    vx = (rng.standard_normal((1, 1, n + T, D)) * 2.0 ** (12 * grow / 9)).astype(np.float32)
    k, v = ((_pack(kx, bits), _pack(vx, bits)) if bits else (_bf(kx), _bf(vx)))
    words = ref.ancestors(_trees(rng, 1, T))[0]
    _check(_attend(q, k, v, [n], words, 0.125, T, bits), q, k, v, [n], words, 0.125, T, bits)


def test_attention_strides_and_views():
    """Queries in token-major order, an output in the same order, a cache that is a slice of a larger one."""
    from myinfer_b200.tree import tree_attention
    rng = np.random.default_rng(3)
    B, Hq, Hk, L, D, bits = 2, 8, 2, 5, 128, 8
    rows, lengths = 90, [40, 77]
    k, v = _cache(rng, B + 1, Hk + 1, rows + 7, D, bits), _cache(rng, B + 1, Hk + 1, rows + 7, D, bits)
    cut = lambda t: tuple(x.cuda()[1:, 1:, 3:3 + rows] for x in t)  # noqa: E731
    tok = _bf(rng.standard_normal((B, L, Hq, D))).cuda()
    q = tok.transpose(1, 2)
    words = ref.ancestors(_trees(rng, B, L))[0]
    store = torch.full((B, L, Hq, D), math.nan, dtype=torch.bfloat16, device="cuda")
    n = torch.tensor(lengths, dtype=torch.int32).cuda()
    anc = torch.from_numpy(words.view(np.int64).copy()).cuda()
    out = tree_attention(q, cut(k), cut(v), n, anc, D ** -0.5, bits=bits, out=store.transpose(1, 2))
    assert out.data_ptr() == store.data_ptr()
    kc, vc = (tuple(x[1:, 1:, 3:3 + rows] for x in t) for t in (k, v))
    _check(out, q, kc, vc, lengths, words, D ** -0.5, L, bits)
    odd = torch.empty(q.numel() + 1, dtype=torch.bfloat16, device="cuda")[1:].view(q.shape).copy_(q)  # 2-byte aligned
    assert torch.equal(out, tree_attention(odd, cut(k), cut(v), n, anc, D ** -0.5, bits=bits))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = tree_attention(q, cut(k), cut(v), n, anc, D ** -0.5, bits=bits)
    s.synchronize()
    assert torch.equal(out, other)


def test_attention_capacity_and_odd_heads():
    """A tree that would pass the cache's end sees what is there; head starts at odd rows (scales 2-byte aligned)."""
    rng = np.random.default_rng(8)
    for D, bits in ((64, 8), (64, 4), (128, 4), (64, 0)):
        B, Hq, Hk, L, rows = 1, 6, 3, 6, 141
        q = _bf(rng.standard_normal((B, Hq, L, D))).cuda()
        k, v = _cache(rng, B, Hk, rows, D, bits), _cache(rng, B, Hk, rows, D, bits)
        words = ref.ancestors(_trees(rng, B, L))[0]
        for n in (138, 141):
            _check(_attend(q, k, v, [n], words, D ** -0.5, L, bits), q, k, v, [n], words, D ** -0.5, L, bits)


def test_attention_strides_of_single_dimensions():
    """A dimension of size 1 may have any stride: batch, kv heads and rows of one."""
    from myinfer_b200.tree import tree_attention
    rng = np.random.default_rng(12)
    for bits in (0, 4, 8):
        for rows in (1, 70):
            k, v = _cache(rng, 1, 1, rows, 64, bits), _cache(rng, 1, 1, rows, 64, bits)
            odd = lambda t: t.as_strided(t.shape, (7, 5, 3 if rows == 1 else t.shape[3], 1))  # noqa: E731
            cut = lambda t: tuple(odd(x.cuda()) for x in t) if bits else odd(t.cuda())  # noqa: E731
            q = _bf(rng.standard_normal((1, 3, 1, 64))).cuda()
            n = torch.tensor([rows - 1], dtype=torch.int32).cuda()
            anc = torch.ones(1, 1, dtype=torch.int64).cuda()
            out = tree_attention(q, cut(k), cut(v), n, anc, 0.125, bits=bits)
            _check(out, q, k, v, [rows - 1], np.ones((1, 1), np.uint64), 0.125, 1, bits)


def test_attention_far_offsets():
    """A head that starts more than 2^31 bytes and 2^30 elements into the cache."""
    from myinfer_b200.tree import tree_attention
    rng = np.random.default_rng(9)
    D, rows, n, L = 128, 9_000_000, 300, 4
    q = _bf(rng.standard_normal((1, 4, L, D))).cuda()
    small = [_cache(rng, 1, 2, n + L, D, 0) for _ in range(2)]
    big = []
    for t in small:
        x = torch.empty(1, 2, rows, D, dtype=torch.bfloat16, device="cuda")
        x[:, :, :n + L] = t.cuda()
        big.append(x)
    words = ref.ancestors(_trees(rng, 1, L))[0]
    out = tree_attention(q, big[0], big[1], torch.tensor([n], dtype=torch.int32).cuda(),
                         torch.from_numpy(words.view(np.int64).copy()).cuda(), D ** -0.5, bits=0)
    _check(out, q, small[0], small[1], [n], words, D ** -0.5, L, 0)


def test_attention_in_a_graph():
    """Captured once, replayed with other lengths: nothing of the call lives on the host."""
    from myinfer_b200.tree import tree_attention
    rng = np.random.default_rng(10)
    L, D, bits = 5, 128, 4
    q = _bf(rng.standard_normal((2, 8, L, D))).cuda()
    k, v = _cache(rng, 2, 2, 600, D, bits), _cache(rng, 2, 2, 600, D, bits)
    kc, vc = _cuda(k), _cuda(v)
    words = ref.ancestors(_trees(rng, 2, L))[0]
    n = torch.tensor([10, 300], dtype=torch.int32).cuda()
    anc = torch.from_numpy(words.view(np.int64).copy()).cuda()
    tree_attention(q, kc, vc, n, anc, 0.09, bits=bits)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = tree_attention(q, kc, vc, n, anc, 0.09, bits=bits)
    for lengths in ([10, 300], [595, 0], [64, 65]):
        n.copy_(torch.tensor(lengths, dtype=torch.int32))
        g.replay()
        torch.cuda.synchronize()
        _check(out, q, k, v, lengths, words, 0.09, L, bits)


def test_plan():
    from myinfer_b200.tree import tree_plan
    rng = np.random.default_rng(1)
    for B, T in ((1, 1), (3, 2), (5, 33), (2, 64)):
        p = _trees(rng, B, T)
        if T > 20:
            p[0, 9] = -1            # a second root
            p[1, 7] = 7             # no earlier node: 7 and what hangs below it are no nodes
            p[1, 15] = 7
            p[1, 16] = 15
            p[1, 17:20] = (40, -5, 19)
        anc, depth = tree_plan(torch.from_numpy(p).cuda())
        bits, d = ref.ancestors(p)
        assert (anc.cpu().numpy().view(np.uint64) == bits).all() and (depth.cpu().numpy() == d).all()
    chain = np.arange(-1, 63, dtype=np.int32)[None]
    anc, depth = tree_plan(torch.from_numpy(chain).cuda())
    assert anc[0, 63].item() == -1 and depth[0, 63].item() == 63


def _logits_inputs(rng, B, T, V, dtype, n_bias, mask):
    R = B * T
    x = (3 * rng.standard_normal((R, V))).astype(np.float32)
    x = torch.from_numpy(x).to(dtype)
    counts = (rng.random((B, V)) < 0.2) * rng.integers(1, 5, (B, V))
    pen = np.stack([1 + rng.random(B), rng.random(B) - 0.3, rng.random(B)], 1).astype(np.float32)
    words = ref.ancestors(_trees(rng, B, T))[0]
    tok = rng.integers(0, V, (B, T)).astype(np.int32)
    if T > 3:
        tok[:, T - 1] = tok[:, 0]   # a token twice on a path
        tok[0, 1] = -1              # and none at all
    ids = rng.integers(0, V, (B, n_bias)).astype(np.int32)
    if n_bias > 4:
        ids[:, -1] = ids[:, 0]      # the last entry of a token counts
        ids[:, 2] = -1
        ids[:, 3] = V
        ids[0, 4] = tok[0, 0]       # a bias on a path's token
    val = (4 * rng.standard_normal((B, n_bias))).astype(np.float32)
    m = None
    if mask:
        m = rng.integers(-2 ** 31, 2 ** 31 - 1, (R, (V + 31) // 32)).astype(np.int32)
        m[0] = 0                    # nothing left
        if R > 1:
            m[1] = -1
    return x, counts.astype(np.int32), pen, tok, words, ids, val, m


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,T,V,n_bias,mask", [(1, 1, 1, 0, False), (1, 1, 1000, 0, True), (2, 5, 4099, 40, True),
                                               (3, 1, 8191, 7, False), (1, 64, 4096, 300, True),
                                               (2, 3, 40000, 1024, True), (1, 2, 151936, 5, True)])
def test_process_logits(dtype, B, T, V, n_bias, mask):
    """Every operation is one correctly rounded fp32 operation: at most 6 of them,
    2^-24 each of the largest value on the way, then the logits' own rounding: the result lies
    between the roundings of the exact value less and plus that error.  Choices are the first
    largest of the values returned."""
    from myinfer_b200.tree import process_logits
    rng = np.random.default_rng(V + T)
    x, counts, pen, tok, words, ids, val, m = _logits_inputs(rng, B, T, V, dtype, n_bias, mask)
    up = lambda a: None if a is None else torch.from_numpy(a).cuda()  # noqa: E731
    kw = dict(batch=B, counts=up(counts), penalties=up(pen), tokens=up(tok), ancestors=up(words.view(np.int64).copy()),
              mask=up(m))
    if n_bias:
        kw.update(bias_ids=up(ids), bias_values=up(val))
    lg = x.cuda()
    out, choice = process_logits(lg, **kw)
    assert out.dtype == dtype and torch.equal(lg.cpu(), x)
    got, pick = _f64(out), choice.cpu().numpy()
    rounded = lambda z: _f64(torch.from_numpy(z).to(dtype))  # noqa: E731
    for r in range(B * T):
        b, t = divmod(r, T)
        path = [tok[b, j] for j in range(T) if int(words[b, t]) >> j & 1]
        want = ref.process_row(_f64(x[r]), counts[b], pen[b], path, list(zip(ids[b], val[b])),
                               None if m is None else m[r].view(np.uint32))
        gone = np.isneginf(want)
        assert (np.isneginf(got[r]) == gone).all()
        big = 2 * np.abs(_f64(x[r])) + 1 + counts[b].astype(np.float64) + T + (np.abs(val[b]).max() if n_bias else 0)
        e, y = 6 * 2.0 ** -24 * big[~gone], got[r][~gone]
        assert (rounded(want[~gone] - e) <= y).all() and (y <= rounded(want[~gone] + e)).all(), r
        assert pick[r] == ref.choice(got[r]), r
    inplace, c2 = process_logits(lg, out=lg, **kw)
    assert inplace is lg and torch.equal(lg, out) and torch.equal(c2, choice)


def test_process_logits_division():
    """The repetition penalty's quotient is the correctly rounded one: bit for bit torch's fp32 division, for values
    and penalties of all sizes (subnormal, infinite and zero ones too)."""
    from myinfer_b200.tree import process_logits
    g = torch.Generator(device="cuda").manual_seed(2)
    V = 1 << 16
    for rep in (1.1, 1.0000001, 1.9999999, 0.3, 3.0, 7.5e-7, 1e30, 1e-38, float("inf")):
        bits = torch.randint(0, 0x7F800001, (4, V), generator=g, device="cuda", dtype=torch.int32)
        x = bits.view(torch.float32)
        x[1] = 30 * torch.rand(V, generator=g, device="cuda")
        x[2] = torch.randn(V, generator=g, device="cuda").abs() * 2.0 ** -100
        x[3] = torch.rand(V, generator=g, device="cuda") + 1.0
        x[0, :3] = torch.tensor([0.0, math.inf, 1.0])
        counts = torch.ones(4, V, dtype=torch.int32, device="cuda")
        pen = torch.tensor([[rep, 0.0, 0.0]] * 4, device="cuda")
        out, _ = process_logits(x, counts=counts, penalties=pen)
        want = x / pen[:, :1]
        assert torch.equal(out.nan_to_num(nan=-1.0), want.nan_to_num(nan=-1.0)), rep


def test_process_logits_strides_nan_and_ties():
    from myinfer_b200.tree import process_logits
    V = 5003
    store = torch.full((3, V + 13), 7.0, dtype=torch.bfloat16, device="cuda")
    lg = store[:, 5:5 + V]
    lg.copy_(torch.zeros(3, V))
    lg[0, 100], lg[0, 4000] = 2.0, 2.0             # a tie: the lowest index
    lg[0, 50] = math.nan                           # never chosen
    lg[1, 3] = -0.0
    lg[1, :3] = -1.0                               # -0 ties with 0
    lg[2] = math.nan
    lg[2, 4999] = -3.0
    out, c = process_logits(lg, out=lg)
    assert c.tolist() == [100, 3, 4999] and out.data_ptr() == lg.data_ptr()
    assert (store[:, :5] == 7).all() and (store[:, 5 + V:] == 7).all()
    m = torch.full((3, (V + 31) // 32), -1, dtype=torch.int32, device="cuda")
    m[0, 50 // 32] = 0                             # NaN and infinity in masked places
    m[2] = 0
    lg[2, 7] = math.inf
    out, c = process_logits(lg, mask=m)
    assert c.tolist() == [100, 3, -1] and not torch.isnan(out[0]).any() and torch.isneginf(out[2]).all()
    lg[1, 17] = math.inf
    assert process_logits(lg)[1][1].item() == 17
    one, c = process_logits(lg[:1])                # one row of a wider tensor
    assert c.item() == 100 and one.shape == (1, V)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_process_logits_parts_without_work(dtype):
    """The choice is joined over a row's CTAs, whichever starts or ends first: all but one part masked out (their CTAs
    load nothing), rows of one part, and calls close behind one another on two streams."""
    from myinfer_b200.tree import process_logits
    g = torch.Generator(device="cuda").manual_seed(6)
    for R, V in ((1, 65536), (1, 65541), (3, 4097), (40, 12000)):
        x = torch.randn(R, V, generator=g, device="cuda").to(dtype)
        streams = [torch.cuda.Stream() for _ in range(2)]
        masks, want = [], []
        for part in range(16):
            lo, hi = part * V // 16, (part + 1) * V // 16
            keep = torch.zeros(R, (V + 31) // 32 * 32, dtype=torch.int64, device="cuda")
            keep[:, lo:hi] = 1
            m = (keep.view(R, -1, 32) << torch.arange(32, device="cuda")).sum(-1)
            masks.append(m.to(torch.uint32).view(torch.int32))
            want.append(lo + x[:, lo:hi].float().argmax(1).to(torch.int32))
        torch.cuda.synchronize()
        got = []
        for i in range(64):
            with torch.cuda.stream(streams[i & 1]):
                got.append(process_logits(x, mask=masks[i % 16])[1])
        torch.cuda.synchronize()
        for i, c in enumerate(got):
            assert torch.equal(c, want[i % 16]), (R, V, i)


def test_process_logits_matches_greedy_sampler_without_processors():
    from myinfer_b200 import ops
    from myinfer_b200.tree import process_logits
    x = torch.randn(1, 151936, device="cuda").to(torch.bfloat16)
    out, c = process_logits(x)
    assert torch.equal(out, x) and c.item() == ops.argmax(x[0]).item()


@pytest.mark.parametrize("B,T", [(1, 1), (2, 2), (9, 17), (64, 64)])
def test_accept(B, T):
    from myinfer_b200.tree import tree_accept
    rng = np.random.default_rng(T)
    V = 50
    p = _trees(rng, B, T)
    tok = rng.integers(0, 6, (B, T)).astype(np.int32)   # few tokens: siblings with the same one
    pick = rng.integers(0, 6, (B, T)).astype(np.int32)
    if T > 5:
        p[0, T - 2:] = -2                                # padding
        pick[1, 0] = 49                                  # nothing accepted
        p[-1], tok[-1], pick[-1] = np.arange(-1, T - 1), 3, 3  # a chain accepted to its end
    counts = rng.integers(0, 9, (B, V)).astype(np.int32)
    dev = [torch.from_numpy(a.copy()).cuda() for a in (p, tok, pick, counts)]
    path, n, nxt = tree_accept(*dev[:3], counts=dev[3])
    for b in range(B):
        want, follow = ref.accept(p[b], tok[b], pick[b])
        assert n[b].item() == len(want) and nxt[b].item() == follow
        assert path[b].tolist() == want + [-1] * (T - len(want))
        for i in want:
            counts[b, tok[b, i]] += 1
    assert (dev[3].cpu().numpy() == counts).all()
    assert torch.equal(tree_accept(*dev[:3])[0], path)


@pytest.mark.parametrize("bits", [0, 4, 8])
@pytest.mark.parametrize("D", [64, 128])
def test_commit(bits, D):
    from myinfer_b200.tree import CacheLayers, commit_tree
    rng = np.random.default_rng(bits + D)
    B, Hk, rows, T = 3, 2, 133, 64
    path = np.full((B, T), -1, np.int32)
    lens = np.array([0, 69, 75], np.int32)               # the last one's tree passes the end of the cache
    for b, p in enumerate(([0, 1, 4, 5, 9, 63], list(range(64)), [0, 2, 40, 57, 58, 60])):
        path[b, :len(p)] = p
    n = np.array([6, 64, 6], np.int32)
    layers, before = [], []
    for _ in range(130):                                 # more layers than one launch takes
        pair = []
        for _ in range(2):
            if bits:
                pair.append((torch.randint(-2 ** 31, 2 ** 31 - 1, (B, Hk, rows, D * bits // 32), dtype=torch.int32,
                                           device="cuda"),
                             *[torch.randn(B, Hk, rows, D // 64, device="cuda").to(torch.bfloat16) for _ in range(2)]))
            else:
                pair.append(torch.randn(B, Hk, rows, D, device="cuda").to(torch.bfloat16))
        layers.append(tuple(pair))
        before.append([x.clone() for t in pair for x in (t if bits else (t,))])
    table = CacheLayers(layers)
    args = [torch.from_numpy(a).cuda() for a in (lens, path, n)]
    commit_tree(table, *args)
    for (k, v), old in zip(layers, before):
        for x, o in zip((*k, *v) if bits else (k, v), old):
            want = o.clone()
            for b in range(B):
                for i in range(n[b]):
                    if lens[b] + max(path[b, i], i) < rows:
                        want[b, :, lens[b] + i] = o[b, :, lens[b] + path[b, i]]
            assert torch.equal(x, want)


def test_refusals():
    from myinfer_b200 import tree
    dev = "cuda"
    q = torch.zeros(1, 4, 2, 128, dtype=torch.bfloat16, device=dev)
    k = torch.zeros(1, 2, 8, 128, dtype=torch.bfloat16, device=dev)
    n = torch.zeros(1, dtype=torch.int32, device=dev)
    a = torch.zeros(1, 2, dtype=torch.int64, device=dev)
    ok = lambda **kw: tree.tree_attention(**{**dict(queries=q, q_keys=k, q_values=k, lengths=n, ancestors=a, scale=1.0,  # noqa: E731
                                                    bits=0), **kw})
    assert ok().shape == q.shape
    wide = torch.zeros(1, 2, 8, 256, dtype=torch.bfloat16, device=dev)[..., :128]
    shifted = torch.zeros(1 * 2 * 8 * 128 + 4, dtype=torch.bfloat16, device=dev)[4:].view(1, 2, 8, 128)
    for kw in (dict(queries=q.float()), dict(queries=q.cpu()), dict(queries=q[..., :96]), dict(q_keys=wide),
               dict(queries=torch.zeros(1, 4, 65, 128, dtype=torch.bfloat16, device=dev)), dict(tree_len=65),
               dict(tree_len=0), dict(q_keys=k[:, :1]), dict(queries=q[:, :3]), dict(lengths=n.long()),
               dict(lengths=torch.zeros(2, dtype=torch.int32, device=dev)), dict(ancestors=a.int()), dict(bits=8),
               dict(bits=3), dict(q_values=k.half()), dict(lengths=n.cpu()), dict(out=torch.empty_like(q).float())):
        with pytest.raises(ValueError):
            ok(**kw)
    from myinfer_b200._lib import M5CudaError
    with pytest.raises(M5CudaError, match="aligned"):
        ok(q_keys=shifted)
    lg = torch.zeros(6, 100, dtype=torch.bfloat16, device=dev)
    for kw in (dict(batch=4), dict(counts=torch.zeros(6, 100, dtype=torch.int32, device=dev)),
               dict(bias_ids=torch.zeros(6, 1, dtype=torch.int32, device=dev)),
               dict(mask=torch.zeros(6, 3, dtype=torch.int64, device=dev)), dict(out=lg.float()),
               dict(tokens=torch.zeros(6, 1, dtype=torch.int32, device=dev))):
        with pytest.raises(ValueError):
            tree.process_logits(lg, **kw)
    for bad in (lg.half(), lg.cpu(), lg.t(), lg[0]):
        with pytest.raises(ValueError):
            tree.process_logits(bad)
    with pytest.raises(M5CudaError, match="mask"):
        tree.process_logits(lg, mask=torch.zeros(6, 3, dtype=torch.int32, device=dev))
    p = torch.zeros(2, 5, dtype=torch.int32, device=dev)
    for bad in (p.cpu(), p.long(), p[0], torch.zeros(1, 65, dtype=torch.int32, device=dev)):
        with pytest.raises(ValueError):
            tree.tree_plan(bad)
    with pytest.raises(ValueError):
        tree.tree_accept(p, p[:, :4].contiguous(), p)
    with pytest.raises(ValueError):
        tree.tree_accept(p, p, p, counts=torch.zeros(3, 9, dtype=torch.int32, device=dev))
    for bad in ([], [(wide, wide)], [(k, k[:, :, :4])], [(k.half(), k.half())], [(k, k), (k[:, :1].contiguous(),) * 2]):
        with pytest.raises(ValueError):
            tree.CacheLayers(bad)
    with pytest.raises(ValueError):
        tree.commit_tree([(k, k)], n, p, n)


@pytest.mark.parametrize("bits", [0, 4, 8])
@pytest.mark.parametrize("keys", ["zero", "tiny", "last tile zero", "any"])
@pytest.mark.parametrize("n,T", [(0, 1), (5, 2), (64, 5), (70, 3), (1024, 7), (1000, 64)])
def test_attention_zero_queries_and_keys(n, T, keys, bits):
    """A query of zeros weighs all keys alike, and so do keys of zeros: in tiles with hidden keys, in tiles that hide
    all of theirs (tree keys that the row does not see, behind a whole tile), in runs that are cut."""
    rng = np.random.default_rng(n + T)
    for D, Hq in ((64, 2), (128, 20)):
        q = 1.5 * rng.standard_normal((1, Hq, T, D))
        q[:, ::2] = 0
        q[:, 1, 0] = 1e-36
        x = rng.standard_normal((1, 1, n + T, D)).astype(np.float32)
        x *= dict(zero=0.0, tiny=1e-36).get(keys, 1.0)
        if keys == "last tile zero":
            x[:, :, n // 64 * 64:] = 0
        q, k = _bf(q).cuda(), (_pack(x, bits) if bits else _bf(x))
        v = _cache(rng, 1, 1, n + T, D, bits)
        for words in (ref.ancestors(_trees(rng, 1, T))[0], np.zeros((1, T), np.uint64)):
            _check(_attend(q, k, v, [n], words, D ** -0.5, T, bits), q, k, v, [n], words, D ** -0.5, T, bits)


@pytest.mark.parametrize("bits", [0, 4, 8])
@pytest.mark.parametrize("n", [0, 40, 3000])
@pytest.mark.parametrize("T", [4, 40])
def test_attention_queries_without_a_number(T, n, bits):
    """What the softmax makes no number of is NaN, in runs that one CTA ends and in runs that are cut: a query with NaN
    or an infinity, scores that are all -inf, a scale of NaN.  A query that sees nothing gives zeros whatever it
    holds, and the other queries of the call what they give without it."""
    rng = np.random.default_rng(T)
    D, Hq = 128, 4
    q = _bf(rng.standard_normal((1, Hq, T, D)))
    k, v = _cache(rng, 1, 1, n + T, D, bits), _cache(rng, 1, 1, n + T, D, bits)
    words = np.array([[(1 << (i + 1)) - 1 for i in range(T)]], np.uint64)  # a chain
    clean = _attend(q.cuda(), k, v, [n], words, 0.1, T, bits)
    bad = q.clone()
    bad[0, 0, 1, 3] = math.nan
    bad[0, 1, 1, 5] = math.inf
    bad[0, 2, 3] = math.nan
    out = _attend(bad.cuda(), k, v, [n], words, 0.1, T, bits)
    rows = torch.zeros(1, Hq, T, dtype=torch.bool)
    rows[0, 0, 1] = rows[0, 1, 1] = rows[0, 2, 3] = True
    assert torch.isnan(out[rows]).all() and torch.equal(out[~rows], clean[~rows])
    assert torch.isnan(_attend(q.cuda(), k, v, [n], words, math.nan, T, bits)).all()
    k0 = k.clone() if bits == 0 else tuple(t.clone() for t in k)
    if bits:
        k0[1].fill_(0.0)
        k0[2].fill_(2.0)   # every key is 2 in all dims
    else:
        k0.fill_(2.0)
    low = q.clone()
    low[0, 3, 2, 7] = -math.inf
    out = _attend(low.cuda(), k0, v, [n], words, 0.1, T, bits)
    assert torch.isnan(out[0, 3, 2]).all() and torch.isfinite(out[0, :3]).all()
    if n == 0:
        words[0, 1] = words[0, 2] = 0
        for x, kk in ((bad, k), (low, k0)):
            assert (_attend(x.cuda(), kk, v, [n], words, 0.1, T, bits)[0, :, 1:3] == 0).all()


@pytest.mark.parametrize("bits", [0, 4, 8])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("heads", [1, 20])
def test_attention_broken_node(heads, bad, bits):
    """A node whose key or value holds NaN or an infinity spoils the queries that see it and no others: their
    results are those of a run in which its row is zero, whatever shares the tile, the run or the call with it."""
    rng = np.random.default_rng(heads)
    B, Hk, T, D, node = 2, 2, 8, 128, 2
    for lengths in ([130, 5], [60, 127], [2000, 640]):
        q = _bf(rng.standard_normal((B, Hk * heads, T, D))).cuda()
        k, v = (_cache(rng, B, Hk, max(lengths) + T, D, bits) for _ in range(2))
        words = ref.ancestors(_trees(rng, B, T))[0]
        sees = torch.zeros(B, T, dtype=torch.bool)
        sees[0] = torch.from_numpy((words[0] >> np.uint64(node) & np.uint64(1)).astype(bool))
        assert 0 < sees[0].sum() < T
        at = (0, slice(None), lengths[0] + node)
        for which in (0, 1):
            kv = [tuple(x.clone() for x in t) if bits else t.clone() for t in (k, v)]
            for x in kv[which] if bits else (kv[which],):
                x[at] = 0
            want = _attend(q, *kv, lengths, words, 0.1, T, bits).transpose(1, 2).cpu()
            for part in (kv[which][1:] if bits else (kv[which],)):   # a group's scale, its bias; one element
                part[(*at, 1 if bits else 77)] = bad
                out = _attend(q, *kv, lengths, words, 0.1, T, bits).transpose(1, 2).cpu()
                assert torch.equal(out[~sees], want[~sees]), (which, lengths)
                if which or math.isnan(bad):                          # an infinite key may weigh nothing
                    assert not torch.isfinite(out[sees]).all(-1).any(), (which, lengths)
                part[(*at, 1 if bits else 77)] = 0


@pytest.mark.parametrize("bits", [0, 4, 8])
def test_attention_broken_committed_key(bits):
    """All queries see a committed key.  NaN in K gives NaN, NaN in V at least in the elements that hold it; a score of
    -inf weighs nothing and leaves the other keys' weights as they are."""
    rng = np.random.default_rng(4)
    Hk, T, D, n = 2, 3, 128, 700
    q = _bf(np.abs(rng.standard_normal((1, 4, T, D)))).cuda()
    k, v = (_cache(rng, 1, Hk, n + T, D, bits) for _ in range(2))
    words = ref.ancestors(_trees(rng, 1, T))[0]

    def put(t, value, at):
        t = tuple(x.clone() for x in t) if bits else t.clone()
        if bits:
            t[1][0, :, at, 0] = 0.0      # scale 0, bias the value: the whole first group
            t[2][0, :, at, 0] = value
        else:
            t[0, :, at, :64] = value
        return t

    def without(t, at):
        cut = lambda x: torch.cat([x[:, :, :at], x[:, :, at + 1:]], 2)  # noqa: E731
        return tuple(cut(x) for x in t) if bits else cut(t)
    for at in (10, 64 * 5 + 63, n - 1):
        assert torch.isnan(_attend(q, put(k, math.nan, at), v, [n], words, 0.05, T, bits)).all()
        out = _attend(q, k, put(v, math.nan, at), [n], words, 0.05, T, bits)
        assert torch.isnan(out[..., :64]).all()
        out = _attend(q, put(k, -math.inf, at), v, [n], words, 0.05, T, bits)
        _check(out, q, without(k, at), without(v, at), [n - 1], words, 0.05, T, bits)


@pytest.mark.parametrize("change", ["reserve", "quantize", "list"])
def test_commit_follows_a_reallocated_cache(change):
    """A table of a cache whose buffers have moved since it was made: the rows move in the buffers of now."""
    from myinfer_b200.cache import KVCache, PromptCache
    from myinfer_b200.tree import CacheLayers, commit_tree
    g = torch.Generator(device="cuda").manual_seed(1)
    layers = [KVCache(2, 128, "cuda", 256) for _ in range(3)]
    cache = layers if change == "list" else PromptCache(layers, "cuda")
    for c in cache:
        c.update_and_fetch(*(torch.randn(1, 2, 40, 128, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2)))
    table = CacheLayers(cache)
    args = [torch.tensor(x, dtype=torch.int32).cuda() for x in ([30], [[0, 2, 5, -1, -1, -1]], [3])]
    for i, c in enumerate(cache):
        if change == "quantize":
            cache[i] = c.to_quantized(64, 8)
        else:
            c.reserve(1000)
    old = [[x.clone() for x in c._tensors()] for c in cache]
    commit_tree(table, *args)
    for c, before in zip(cache, old):
        for x, o in zip(c._tensors(), before):
            o[:, :, 31], o[:, :, 32] = o[:, :, 32].clone(), o[:, :, 35].clone()
            assert torch.equal(x, o)


def test_commit_refuses_a_cache_without_buffers():
    from myinfer_b200.cache import KVCache, PromptCache
    from myinfer_b200.tree import CacheLayers
    with pytest.raises(ValueError, match="without buffers"):
        CacheLayers(PromptCache([KVCache(2, 128, "cuda")], "cuda"))
    with pytest.raises(ValueError, match="no cache layers"):
        CacheLayers(PromptCache([], "cuda"))


@pytest.mark.parametrize("bits", [0, 4, 8])
@pytest.mark.parametrize("n", [500, 9000])
def test_attention_shrinking_values(bits, n):
    """Values of 2^12 first, at keys that weigh nothing, and of 1 behind them.  In fp16 a value is off by u of itself
    or, far below the largest of its run so far, by half a subnormal unit, 2^-25.  The largest is held at 2^-3 or more
    for codes, whose bias is rounded too (2 x 2^-22 of the largest), and at 2^7 or more for bf16 (2^-32)."""
    rng = np.random.default_rng(13)
    L = T = 3
    D, big, first = 64, 2.0 ** 12, 20
    q = np.abs(rng.standard_normal((1, 2, L, D))) + 0.5
    kx = rng.standard_normal((1, 1, n + T, D)).astype(np.float32)
    kx[:, :, :first] = -6.0                      # scores below the others' by hundreds
    vx = rng.standard_normal((1, 1, n + T, D)).astype(np.float32)
    vx[:, :, :first] *= big
    q = _bf(q).cuda()
    k, v = ((_pack(kx, bits), _pack(vx, bits)) if bits else (_bf(kx), _bf(vx)))
    words = ref.ancestors(_trees(rng, 1, T))[0]
    out = _f64(_attend(q, k, v, [n], words, 0.25, T, bits))
    kd, vd = _dense(k, bits), _dense(v, bits)
    want, mag = ref.attention(_f64(q)[0], kd[0], vd[0], n, words[0], T, 0.25)
    if bits:
        s, b = _f64(v[1]), _f64(v[2])
        unit = 2.0 ** -21 * max(np.abs(b).max(), np.abs(s * (2 ** bits - 1) + b).max())
    else:
        unit = 2.0 ** -32 * np.abs(vd).max()
    for h in range(2):
        d = 8 / math.sqrt(3) * U * 0.25 * np.sqrt((_f64(q)[0, h] ** 2) @ (kd[0, 0] ** 2).T).max(1)
        tol = 2.0 ** -8 * np.abs(want[h]) + unit + (np.expm1(2 * d) + 4 * U)[:, None] * mag[h]
        err = np.abs(out[0, h] - want[h])
        assert (err <= tol).all(), float((err - tol).max())
