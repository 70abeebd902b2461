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
from typing import List, Optional, Sequence, Tuple, Union

import torch

from . import _lib
from ._lib import M5LayerKv

MAX_NODES = 64

_Kv = Union[torch.Tensor, Sequence[torch.Tensor]]
_ENTRIES = ("m5_tree_plan", "m5_tree_attention_workspace", "m5_tree_attention", "m5_process_logits", "m5_tree_accept",
            "m5_tree_commit")
_calls = None


def _load():
    """The compiled entries (csrc/tree_binding.cpp: argument checks, results, the call), over libm5cuda's operators."""
    global _calls
    L = _lib.lib()
    try:
        from . import _tree_binding
    except ImportError as e:
        raise _lib.M5CudaError(_lib.M5_ERR_STATE, f"_tree_binding.so: {e}; run `python -m myinfer_b200.build`") from e
    _tree_binding.bind(*(ctypes.cast(getattr(L, n), ctypes.c_void_p).value for n in _ENTRIES), _lib.check)
    _calls = _tree_binding
    return _calls


def tree_plan(parents: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """(ancestors int64 [B, T], depths int32 [B, T]) of trees given by int32
    ``parents`` [B, T] (-1: a root).  Bit j of ``ancestors[b, i]`` is set where
    j is i or above it.  Nodes that belong to no tree (a parent that is neither
    -1 nor an earlier node, and everything below) get 0."""
    return (_calls or _load()).plan(parents)


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
    key gives zeros; a key or value with NaN or an infinity spoils the queries
    that see it, no others.  Returns bf16 [B, Hq, L, D] (``out`` if given)."""
    return (_calls or _load()).attention(queries, q_keys, q_values, lengths, ancestors, scale, tree_len, group_size, bits, out)


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
    return (_calls or _load()).logits(logits, batch, counts, penalties, tokens, ancestors, bias_ids, bias_values, mask, out)


def tree_accept(parents: torch.Tensor, tokens: torch.Tensor, picks: torch.Tensor,
                counts: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(path int32 [B, T], accepted int32 [B], next int32 [B]): from node 0, the
    first child whose ``tokens`` entry equals ``picks`` (the model's choice
    after each node, int32 [B, T]) of its parent, while there is one.  ``path``
    holds the nodes passed (-1 behind them), ``next`` the choice after the last.
    ``counts`` (int32 [B, V], see ``process_logits``) gains 1 for every accepted
    node's token."""
    return (_calls or _load()).accept(parents, tokens, picks, counts)


class CacheLayers:
    """Table of a cache's buffers for ``commit_tree``: a ``PromptCache`` (or a list
    of its layers), whose buffers it follows when they are reallocated or quantized,
    or (keys, values) per layer with the shapes ``tree_attention`` takes (buffers
    contiguous; these very tensors, which the table keeps alive)."""

    def __init__(self, layers):
        # the list and what it held: layers and the generations of their buffers
        self._source = layers if isinstance(layers, list) and all(hasattr(c, "generation") for c in layers) else None
        self._fill(layers)

    def current(self) -> tuple:
        """``call``, after filling the table again if the cache's buffers have moved."""
        src = self._source
        if src is not None and (self._layers != src or self._generations != [c.generation for c in src]):
            self._fill(src)
        return self.call

    def _fill(self, layers):
        pairs: List[tuple] = [(c.keys, c.values) if hasattr(c, "keys") else tuple(c) for c in layers]
        if not pairs:
            raise ValueError("no cache layers")
        arr = (M5LayerKv * len(pairs))()
        shape = None
        for a, (k, v) in zip(arr, pairs):
            if k is None or v is None:
                raise ValueError("a cache layer without buffers")
            packed = not isinstance(k, torch.Tensor)
            ks, vs = (tuple(k), tuple(v)) if packed else ((k,), (v,))
            data = ks[0]
            for t in ks + vs:
                if not t.is_cuda or t.device != data.device or not t.is_contiguous() or t.dim() != 4 or \
                        t.shape[:3] != data.shape[:3]:
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
        self.structs, self._keep = arr, pairs  # the table holds addresses only
        self.call = (ctypes.addressof(arr), len(arr), self.batch, self.kv_heads, self.head_dim, self.device.index)
        if self._source is not None:
            self._layers, self._generations = list(layers), [c.generation for c in layers]


def commit_tree(layers, lengths: torch.Tensor, path: torch.Tensor, accepted: torch.Tensor) -> None:
    """Keep an accepted path (``tree_accept``): in every layer, row ``lengths[b]
    + path[b, i]`` of K and V becomes row ``lengths[b] + i``, i < accepted[b], in
    place.  ``layers``: a ``CacheLayers`` (a loop keeps one), or what it takes; a
    captured graph keeps the buffers of its capture.
    ``lengths`` is left to the caller to advance."""
    t = layers if isinstance(layers, CacheLayers) else CacheLayers(layers)
    (_calls or _load()).commit(*t.current(), lengths, path, accepted)
