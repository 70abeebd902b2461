"""Speculative decoding over a tree of drafted tokens: the operators one round needs.

A sequence ``b`` has ``lengths[b]`` committed keys in its cache rows; node ``i``
of its drafted tree (at most 64 nodes, parents before children, node 0 the
pending token) has its key and value in row ``lengths[b] + i``.  One round of a
decoding loop (``generate.tree_speculative_generate_step``):

* ``tree_plan``       parents -> the nodes' ancestor words and depths;
* ``tree_attention``  every node attends to the cache and to its own path
                      (inside ``Model.forward_tree``);
* ``process_logits``  penalties, biases and a grammar's mask on the nodes'
                      logits, and the greedy choice of each;
* ``tree_accept``     the longest path of drafts that equal the choices;
* ``commit_tree``     the path's rows moved behind the committed ones.

All take CUDA tensors, run on the current torch stream, and do not
synchronise.  With trees of one node they are the operators of plain batched
decoding of sequences of different lengths.
"""

from __future__ import annotations

import ctypes
from ctypes import c_int64, c_size_t
from functools import lru_cache
from typing import List, Optional, Sequence, Tuple, Union

import torch

from . import _lib
from ._lib import M5KvView, M5LayerKv, check, lib

MAX_NODES = 64

_Kv = Union[torch.Tensor, Sequence[torch.Tensor]]
_Int64x3 = c_int64 * 3
_raw_stream = torch._C._cuda_getCurrentRawStream  # the handle alone: a torch.cuda.Stream object costs 2 us


def _launch(name: str, dev: int, *args) -> None:
    """Call a libm5cuda entry point on device ``dev`` and its current stream (the last argument)."""
    fn = getattr(lib(), name)
    if torch._C._cuda_getDevice() == dev:
        check(fn(*args, _raw_stream(dev)))
    else:
        with torch.cuda.device(dev):
            check(fn(*args, _raw_stream(dev)))


def _whole(t: torch.Tensor, shape: tuple, what: str, dev: int, dtype=torch.int32) -> int:
    """Pointer of a contiguous tensor of this shape and type on device ``dev``."""
    if t.dtype is not dtype or t.shape != shape or t.get_device() != dev or not t.is_contiguous():
        raise ValueError(f"{what} must be a contiguous {dtype} tensor of shape {list(shape)} on cuda:{dev}")
    return t.data_ptr()


def _tree_shape(parents: torch.Tensor) -> Tuple[int, int]:
    if parents.dim() != 2 or parents.dtype is not torch.int32 or not parents.is_cuda or not parents.is_contiguous():
        raise ValueError("parents must be a contiguous int32 CUDA tensor [batch, nodes]")
    B, T = parents.shape
    if not 1 <= T <= MAX_NODES:
        raise ValueError(f"a tree has 1 to {MAX_NODES} nodes, got {T}")
    return B, T


@lru_cache(maxsize=256)
def _workspace_bytes(dev: int, B: int, Hq: int, Hkv: int, L: int, D: int) -> int:
    need = c_size_t(0)
    with torch.cuda.device(dev):
        check(lib().m5_tree_attention_workspace(B, Hq, Hkv, L, D, ctypes.byref(need)))
    return need.value


def tree_plan(parents: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """(ancestors int64 [B, T], depths int32 [B, T]) of trees given by int32
    ``parents`` [B, T] (-1: a root).  Bit j of ``ancestors[b, i]`` is set where
    j is i or above it.  Nodes that belong to no tree (a parent that is neither
    -1 nor an earlier node, and everything below) get 0."""
    B, T = _tree_shape(parents)
    anc = torch.empty(B, T, dtype=torch.int64, device=parents.device)
    depth = torch.empty(B, T, dtype=torch.int32, device=parents.device)
    _launch("m5_tree_plan", parents.get_device(), parents.data_ptr(), B, T, anc.data_ptr(), depth.data_ptr())
    return anc, depth


def _kv_parts(t: _Kv, bits: int, D: int, dev: int, what: str):
    """(view, [batch, kv heads, rows, width]) of a K or V operand over the whole cache."""
    if bits:
        if isinstance(t, torch.Tensor) or len(t) != 3:
            raise ValueError(f"{what} of a quantized cache are (wq, scales, biases)")
        data, s, b = t
        width, dtype = D * bits // 32, torch.int32
    else:
        if not isinstance(t, torch.Tensor):
            raise ValueError(f"{what} of an unquantized cache are one bf16 tensor")
        data, width, dtype = t, D, torch.bfloat16
    shape = data.shape
    if len(shape) != 4 or data.dtype is not dtype or shape[3] != width or data.get_device() != dev:
        raise ValueError(f"{what} must be {dtype} [batch, kv heads, rows, {width}] on cuda:{dev}")
    sb, sh, sr, one = data.stride()
    if one != 1 or sr != width or sh % width or sb % width:
        # a dimension of size 1 may have any stride: it is never stepped over
        nb, nh, nr, nw = shape
        sb, sh = (0 if nb == 1 else sb), (0 if nh == 1 else sh)
        if (one != 1 and nw > 1) or (sr != width and nr > 1) or sh % width or sb % width:
            raise ValueError(f"{what}: a head's rows must be contiguous")
    rows_b, rows_h = sb // width, sh // width
    if not bits:
        return M5KvView(data.data_ptr(), None, None, rows_b, rows_h), shape
    G = D // 64
    want, lay = (*shape[:3], G), (rows_b * G, rows_h * G, G, 1)
    for x in (s, b):
        if x.dtype is not torch.bfloat16 or x.shape != want or x.get_device() != dev:
            raise ValueError(f"{what}: scales and biases must be bf16 [batch, kv heads, rows, {G}] on cuda:{dev}")
        if x.stride() != lay and any(n > 1 and a != b for n, a, b in zip(want, x.stride(), lay)):
            raise ValueError(f"{what}: scales and biases must be laid out like the rows")
    return M5KvView(data.data_ptr(), s.data_ptr(), b.data_ptr(), rows_b, rows_h), shape


def tree_attention(queries: torch.Tensor, q_keys: _Kv, q_values: _Kv, lengths: torch.Tensor, ancestors: torch.Tensor,
                   scale: float, tree_len: Optional[int] = None, group_size: int = 64, bits: int = 8,
                   out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """softmax(scale * queries @ K^T) @ V for nodes of drafted trees over a cache.

    queries: bf16 [B, Hq, L, D] (any strides with contiguous dims), L <= 64
    nodes.  q_keys / q_values: the whole cache, MLX tuples ``(wq int32 [B, Hkv,
    rows, D*bits/32], scales, biases)`` or bf16 [B, Hkv, rows, D] with
    ``bits=0``.  lengths: int32 [B] committed keys, seen by every query.
    ancestors: int64 [B, L], bit j = the query sees tree key ``lengths[b] + j``;
    ``tree_len`` (default L) is the number of tree keys.  A query that sees no
    key gives zeros.  Returns bf16 [B, Hq, L, D] (``out`` if given)."""
    if queries.dim() != 4 or queries.dtype is not torch.bfloat16 or not queries.is_cuda:
        raise ValueError("queries must be bf16 CUDA [batch, heads, nodes, dim]")
    B, Hq, L, D = queries.shape
    dev = queries.get_device()
    T = L if tree_len is None else int(tree_len)
    if D not in (64, 128):
        raise ValueError(f"head_dim must be 64 or 128, got {D}")
    if not (1 <= L <= MAX_NODES and 1 <= T <= MAX_NODES):
        raise ValueError(f"a tree has 1 to {MAX_NODES} nodes, got {L} queries and {T} tree keys")
    if bits not in (0, 4, 8) or (bits and group_size != 64):
        raise ValueError("tree_attention supports bits 4/8 with group_size 64, or bits 0 (bf16)")
    kv_k, shape = _kv_parts(q_keys, bits, D, dev, "keys")
    kv_v, vshape = _kv_parts(q_values, bits, D, dev, "values")
    if shape != vshape or shape[0] != B:
        raise ValueError(f"keys {tuple(shape)} and values {tuple(vshape)} must agree and have batch {B}")
    Hkv, rows = shape[1], shape[2]
    if Hkv == 0 or Hq % Hkv:
        raise ValueError("number of query heads must be a multiple of kv heads")
    len_p = _whole(lengths, (B,), "lengths", dev)
    anc_p = _whole(ancestors, (B, L), "ancestors", dev, torch.int64)
    q = queries
    sb, sh, sl, one = q.stride()
    if one != 1 or (sb | sh | sl) % 8 or q.data_ptr() % 16:
        q = q.contiguous()
        if q.data_ptr() % 16:
            q = q.clone()
        sb, sh, sl, one = q.stride()
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif out.shape != queries.shape or out.dtype is not torch.bfloat16 or out.get_device() != dev or out.stride(3) != 1:
        raise ValueError("out must be bf16 of the queries' shape with contiguous dims")
    need = _workspace_bytes(dev, B, Hq, Hkv, L, D)
    # from the stream's own pool: calls on other streams never share it
    ws = torch.empty(need, dtype=torch.uint8, device=q.device)
    _launch("m5_tree_attention", dev, q.data_ptr(), _Int64x3(sb, sh, sl), B, Hq, L, D, kv_k, kv_v, Hkv, rows, len_p, T,
            anc_p, L, float(scale), group_size, bits, out.data_ptr(), _Int64x3(*out.stride()[:3]), ws.data_ptr(), need)
    return out


def process_logits(logits: torch.Tensor, batch: Optional[int] = None, counts: Optional[torch.Tensor] = None,
                   penalties: Optional[torch.Tensor] = None, tokens: Optional[torch.Tensor] = None,
                   ancestors: Optional[torch.Tensor] = None, bias_ids: Optional[torch.Tensor] = None,
                   bias_values: Optional[torch.Tensor] = None, mask: Optional[torch.Tensor] = None,
                   out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Penalties, biases and a grammar's mask on logits [R, V] (bf16 or fp32):
    (processed logits, choices int32 [R]).

    Row ``r`` is node ``r % T`` of sequence ``r // T``, T = R / ``batch`` (default:
    every row its own sequence).  In fp32, rounded once at the end:

    * ``counts`` int32 [batch, V] (times each token has occurred), ``penalties``
      fp32 [batch, 3] = repetition, presence, frequency, and for trees
      ``tokens`` int32 / ``ancestors`` int64 [batch, T], whose tokens on a node's
      own path count too: where c > 0, v < 0 ? v * rep : v / rep, - presence,
      - frequency * c;
    * ``bias_ids`` int32 / ``bias_values`` fp32 [batch, N <= 1024]: added (the last
      entry of a token counts; ids outside the vocabulary are unused);
    * ``mask`` int32 [R, >= ceil(V / 32)]: -inf where bit ``w % 32`` of word
      ``w // 32`` is 0.

    ``choices`` is the first index of a row's largest value, -1 where nothing is
    left.  ``out=logits`` works in place; by default a new tensor is written."""
    if logits.dim() != 2 or logits.dtype not in (torch.bfloat16, torch.float32) or not logits.is_cuda:
        raise ValueError("logits must be bf16 or fp32 CUDA [rows, vocab]")
    R, V = logits.shape
    dev = logits.get_device()
    B = R if batch is None else int(batch)
    if B < 1 or R % B:
        raise ValueError(f"{R} logits rows are no multiple of batch {batch}")
    T = R // B
    if T > MAX_NODES:
        raise ValueError(f"a tree has 1 to {MAX_NODES} nodes, got {T}")
    if logits.stride(1) != 1:
        raise ValueError("logits rows must be contiguous")
    if out is None:
        out = torch.empty_like(logits, memory_format=torch.contiguous_format)
    elif out.shape != logits.shape or out.dtype != logits.dtype or out.device != logits.device or out.stride(1) != 1:
        raise ValueError("out must have the logits' shape and type, with contiguous rows")
    if (counts is not None or tokens is not None) and penalties is None:
        raise ValueError("counts and tokens need penalties")
    if (tokens is None) != (ancestors is None) or (bias_ids is None) != (bias_values is None):
        raise ValueError("tokens come with ancestors, and bias_ids with bias_values")
    cp = None if counts is None else _whole(counts, (B, V), "counts", dev)
    pp = None if penalties is None else _whole(penalties, (B, 3), "penalties", dev, torch.float32)
    tp = None if tokens is None else _whole(tokens, (B, T), "tokens", dev)
    ap = None if ancestors is None else _whole(ancestors, (B, T), "ancestors", dev, torch.int64)
    nb, ip, vp = 0, None, None
    if bias_ids is not None:
        nb = bias_ids.shape[-1]
        ip = _whole(bias_ids, (B, nb), "bias_ids", dev)
        vp = _whole(bias_values, (B, nb), "bias_values", dev, torch.float32)
    mp, mld = None, 0
    if mask is not None:
        mld = mask.shape[-1]
        mp = _whole(mask, (R, mld), "mask", dev)
    choices = torch.empty(R, dtype=torch.int32, device=logits.device)
    # a single row's stride is meaningless (torch keeps any stride on a size-1 dimension)
    ld, old = (logits.stride(0), out.stride(0)) if R > 1 else (V, V)
    dt = _lib.M5_DTYPE_BF16 if logits.dtype is torch.bfloat16 else _lib.M5_DTYPE_F32
    _launch("m5_process_logits", dev, logits.data_ptr(), ld, out.data_ptr(), old, dt, B, T, V, cp, V, pp, tp, ap, ip, vp,
            nb, mp, mld, choices.data_ptr())
    return out, choices


def tree_accept(parents: torch.Tensor, tokens: torch.Tensor, picks: torch.Tensor,
                counts: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(path int32 [B, T], accepted int32 [B], next int32 [B]): from node 0, the
    first child whose ``tokens`` entry equals ``picks`` (the model's choice
    after each node, int32 [B, T]) of its parent, while there is one.  ``path``
    holds the nodes passed (-1 behind them), ``next`` the choice after the last.
    ``counts`` (int32 [B, V], see ``process_logits``) gains 1 for every accepted
    node's token."""
    B, T = _tree_shape(parents)
    dev = parents.get_device()
    tp = _whole(tokens, (B, T), "tokens", dev)
    pp = _whole(picks, (B, T), "picks", dev)
    cp, V = None, 0
    if counts is not None:
        if counts.dim() != 2:
            raise ValueError("counts must be int32 [batch, vocab]")
        V = counts.shape[1]
        cp = _whole(counts, (B, V), "counts", dev)
    path = torch.empty_like(parents)
    n = parents.new_empty(B)
    nxt = torch.empty_like(n)
    _launch("m5_tree_accept", dev, parents.data_ptr(), tp, pp, B, T, path.data_ptr(), n.data_ptr(), nxt.data_ptr(), cp, V, V)
    return path, n, nxt


class CacheLayers:
    """Table of a cache's buffers for ``commit_tree``: a ``PromptCache``, or
    (keys, values) per layer with the shapes ``tree_attention`` takes (buffers
    contiguous).  Build it again when the cache reallocates."""

    def __init__(self, layers):
        pairs: List[tuple] = [(c.keys, c.values) if hasattr(c, "keys") else tuple(c) for c in layers]
        if not pairs:
            raise ValueError("no cache layers")
        self._keep = pairs  # the table holds addresses only
        arr = (M5LayerKv * len(pairs))()
        shape = None
        for a, (k, v) in zip(arr, pairs):
            packed = not isinstance(k, torch.Tensor)
            ks, vs = (tuple(k), tuple(v)) if packed else ((k,), (v,))
            data = ks[0]
            for t in ks + vs:
                if not t.is_cuda or not t.is_contiguous() or t.dim() != 4 or t.shape[:3] != data.shape[:3]:
                    raise ValueError("cache buffers must be contiguous CUDA tensors [batch, kv heads, rows, ...]")
            if packed:
                if len(ks) != 3 or len(vs) != 3 or ks[0].dtype != torch.int32 or vs[0].dtype != torch.int32 or \
                        any(t.dtype != torch.bfloat16 for t in ks[1:] + vs[1:]):
                    raise ValueError("packed cache layers are (int32 words, bf16 scales, bf16 biases)")
                D = ks[1].shape[3] * 64
                bits = ks[0].shape[3] * 32 // D if D else 0
                if bits not in (4, 8) or vs[0].shape != ks[0].shape or \
                        any(t.shape[3] != D // 64 for t in ks[1:] + vs[1:]) or ks[0].shape[3] * 32 != D * bits:
                    raise ValueError("packed cache layers hold 4- or 8-bit codes in groups of 64")
            else:
                D, bits = data.shape[3], 0
                if data.dtype != torch.bfloat16 or vs[0].dtype != torch.bfloat16 or vs[0].shape != data.shape:
                    raise ValueError("unquantized cache layers are bf16 [batch, kv heads, rows, dim]")
            if shape is None:
                shape, self.device = (data.shape[0], data.shape[1], D), data.device
            if (data.shape[0], data.shape[1], D) != shape or data.device != self.device:
                raise ValueError("cache layers differ in batch, heads, head_dim or device")
            a.k, a.v, a.capacity, a.bits, a.group_size = data.data_ptr(), vs[0].data_ptr(), data.shape[2], bits, 64
            if packed:
                a.k_scales, a.k_biases = ks[1].data_ptr(), ks[2].data_ptr()
                a.v_scales, a.v_biases = vs[1].data_ptr(), vs[2].data_ptr()
        self.batch, self.kv_heads, self.head_dim = shape
        if self.head_dim not in (64, 128):
            raise ValueError(f"head_dim must be 64 or 128, got {self.head_dim}")
        self.structs = arr


def commit_tree(layers, lengths: torch.Tensor, path: torch.Tensor, accepted: torch.Tensor) -> None:
    """Keep an accepted path (``tree_accept``): in every layer, row ``lengths[b]
    + path[b, i]`` of K and V becomes row ``lengths[b] + i``, i < accepted[b], in
    place.  ``layers``: a ``CacheLayers`` (a loop keeps one), or what it takes.
    ``lengths`` is left to the caller to advance."""
    t = layers if isinstance(layers, CacheLayers) else CacheLayers(layers)
    if path.dim() != 2 or path.shape[0] != t.batch or not 1 <= path.shape[1] <= MAX_NODES:
        raise ValueError(f"path must be int32 [{t.batch}, 1 to {MAX_NODES} nodes]")
    B, T = path.shape
    dev = t.device.index
    _launch("m5_tree_commit", dev, t.structs, len(t.structs), B, t.kv_heads, t.head_dim,
            _whole(lengths, (B,), "lengths", dev), _whole(path, (B, T), "path", dev), T,
            _whole(accepted, (B,), "accepted", dev))
