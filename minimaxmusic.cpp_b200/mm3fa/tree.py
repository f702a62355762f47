"""Decoding with a tree of drafted tokens (the mm3fa_tree_* entry points of include/mm3fa.h) on torch tensors.

    tree = mm3fa.DraftTree(parents, n_nodes)                     # int32 [n_tree, T], [n_tree]: device memory, read at each call
    layers = mm3fa.CacheLayers(k_caches, v_caches)               # slabs (N, n_head_kv, rows, D) of every layer
    for layer in range(n_layers):
        ...                                                      # the nodes' K and V into rows kv_len + i of the slabs
        out = tree.attend(q, k, v, kv_len, scale)                # each node sees the cache, its ancestors and itself
    path, n_path, token = tree.verify(logits, tokens, accept, sample, draft)      # which nodes stay, and the token after
    kv_len = tree.commit(layers, path, n_path, kv_len)           # their rows together, behind the cache's

Sequence s of N goes by tree s % n_tree (the sets of a CFG batch share theirs).  Every call enqueues on torch's current
stream (or `stream`) of the tensors' device and raises MM3FAError where the C ABI rejects it; nothing synchronises except
`check`.
"""
from __future__ import annotations

import ctypes
import struct

from . import ERR_SHAPE, ERR_STRIDE, ERR_TYPE, MM3FAError, lib
from .ggml import GGML_TYPE_Q8_0, Q8_0_BLOCK_BYTES, QK8_0
from .on_device import _PACK_TENSOR, OnDevice

_PACK_TREE = struct.Struct("@PqP2i").pack  # struct mm3fa_tree

_fns = None


def _calls():
    """The library's entry points with their argument types (structs go in as packed bytes)."""
    global _fns
    if _fns is None:
        L, vp, i, sz, f = lib(), ctypes.c_void_p, ctypes.c_int, ctypes.c_size_t, ctypes.c_float
        sigs = {
            "attn_workspace": (sz, [vp, vp, vp, vp]),
            "attn": (i, [vp, vp, vp, vp, vp, f, f, vp, vp, sz, vp]),
            "verify": (i, [vp, vp, vp, vp, vp, vp, f, vp, vp, vp, vp]),
            "commit": (i, [vp, vp, i, vp, vp, i, i, vp, vp, vp]),
        }
        fns = {}
        for name, (res, args) in sigs.items():
            fn = getattr(L, "mm3fa_tree_" + name)
            fn.restype, fn.argtypes = res, args
            fns[name] = fn
        fns["capture_id"] = fn = L.mm3fa_capture_id
        fn.restype, fn.argtypes = ctypes.c_uint64, [vp]
        _fns = fns
    return _fns


def _slab(t, types, dev, name):
    """mm3fa_tensor [D, rows, heads, sets] of a cache slab (sets, heads, rows, D), or (.., bytes) of Q8_0 blocks as uint8."""
    import torch

    if t.dim() != 4:
        raise MM3FAError(ERR_SHAPE, name + ": a slab has 4 dimensions")
    if t.get_device() != dev:
        raise ValueError(f"{name}: a slab on {t.device}, the others are elsewhere")
    a, b, c, d = t.shape
    sa, sb, sc, sd = t.stride()
    if sd != 1 and d > 1:
        raise MM3FAError(ERR_STRIDE, name + ": a slab's rows have to be contiguous")
    if t.dtype is torch.uint8:
        if d % Q8_0_BLOCK_BYTES:
            raise MM3FAError(ERR_SHAPE, name + ": rows of whole Q8_0 blocks are wanted")
        return _PACK_TENSOR(GGML_TYPE_Q8_0, 0, d // Q8_0_BLOCK_BYTES * QK8_0, c, b, a, Q8_0_BLOCK_BYTES, sc, sb, sa, t.data_ptr())
    ty = types.get(t.dtype)
    if ty is None:
        raise MM3FAError(ERR_TYPE, name)
    ty, e = ty
    return _PACK_TENSOR(ty, 0, d, c, b, a, e, sc * e, sb * e, sa * e, t.data_ptr())


class CacheLayers:
    """The K and V slabs of a cache's layers, for `DraftTree.commit`: one tensor (layers, N, n_head_kv, rows, D) each, or
    lists of (N, n_head_kv, rows, D); F32, F16, BF16, or uint8 with rows of Q8_0 blocks.  The tensors stay the caller's."""

    def __init__(self, k, v):
        from .on_device import _types

        self.k, self.v = list(k), list(v)
        if not self.k or len(self.k) != len(self.v):
            raise MM3FAError(ERR_SHAPE, "CacheLayers")
        self.n_layers, self.device, self.n_seq = len(self.k), self.k[0].device, self.k[0].shape[0]
        types, dev = _types(), self.k[0].get_device()
        self._desc = [b"".join(_slab(t, types, dev, "CacheLayers") for t in x) for x in (self.k, self.v)]


class DraftTree(OnDevice):
    """Trees of up to 256 drafted tokens: parents int32 [n_tree, T], n_nodes int32 [n_tree] or None (T)."""

    _prefix = "mm3fa_tree_"

    def __init__(self, parents, n_nodes=None):
        self._on_device_of(parents)
        if parents.dim() != 2 or parents.shape[0] < 1 or parents.shape[1] < 1:
            raise MM3FAError(ERR_SHAPE, "DraftTree: parents")
        if parents.dtype is not self._int32:
            raise MM3FAError(ERR_TYPE, "DraftTree: parents")
        if parents.shape[1] > 1 and parents.stride(1) != 1:
            raise MM3FAError(ERR_STRIDE, "DraftTree: parents")
        self.parents, self.n_nodes = parents, n_nodes
        self.n_tree, self.max_nodes = parents.shape
        counts = 0 if n_nodes is None else self._ints(n_nodes, self.n_tree, "n_nodes")
        self._desc = _PACK_TREE(parents.data_ptr(), parents.stride(0) if self.n_tree > 1 else self.max_nodes, counts,
                                self.max_nodes, self.n_tree)

    def _calls(self):
        return _calls()

    def _each_node(self, t, dtype, what):
        """Address of a contiguous tensor [n_tree, T]."""
        if t.dtype is not dtype:
            raise MM3FAError(ERR_TYPE, "DraftTree: " + what)
        if t.get_device() != self._dev:
            raise self._elsewhere(t)
        if t.dim() != 2 or t.shape[0] != self.n_tree or t.shape[1] != self.max_nodes:
            raise MM3FAError(ERR_SHAPE, "DraftTree: " + what)
        if not t.is_contiguous():
            raise MM3FAError(ERR_STRIDE, "DraftTree: " + what)
        return t.data_ptr()

    def _rows_of_nodes(self, t, what):
        """mm3fa_tensor [V, T, n_tree, 1] of a tensor (n_tree, T, V)."""
        if t.dim() != 3:
            raise MM3FAError(ERR_SHAPE, "DraftTree: " + what)
        return self._rows(t[None])

    def attend(self, q, k, v, kv_len, scale, out=None, logit_softcap=0.0, ws=None, stream=None):
        """softmax(scale * q k^T) v of the queries q (N, n_head, T, D), where node i of a sequence sees the first kv_len[s]
        rows of its slabs k, v (N, n_head_kv, rows, D), and row kv_len[s] + j for itself and its ancestors j.
        out: (N, T, n_head, D), F32 or q's type; made in q's type when not given, with zeros in the rows of nodes that do
        not count.  ws: a uint8 tensor, its first 64 KiB zero, instead of this object's own workspace of the stream; it serves
        one stream at a time.  (Calls in a capture that torch.cuda.graph has not begun need one.)"""
        if stream is not None:  # what is allocated here belongs to that stream too
            with self._on(stream):
                return self.attend(q, k, v, kv_len, scale, out, logit_softcap, ws)
        qd, st = self._rows(q), self._stream()
        kd, vd = _slab(k, self._dt, self._dev, "DraftTree"), _slab(v, self._dt, self._dev, "DraftTree")
        if out is None:
            make = self._torch.empty if self.n_nodes is None else self._torch.zeros
            out = make((q.shape[0], q.shape[2], q.shape[1], q.shape[3]), dtype=q.dtype, device=q.device)
        if ws is None:
            shape = (q.shape, k.shape, q.dtype, k.dtype)
            need = self._need.get(shape)
            if need is None:
                need = self._need[shape] = self._call("attn_workspace", qd, kd, vd, self._desc)
            ptr, cap = self._workspace(("attn", st), need)
        else:
            ptr, cap = self._given(ws)
        self._run("attn", qd, kd, vd, self._desc, self._ints(kv_len, q.shape[0], "kv_len"), scale, logit_softcap, self._rows(out),
                  ptr, cap, st)
        return out

    def attend_workspace(self, q, k, v) -> int:
        """Bytes of the workspace that `attend` needs for these operands."""
        return self._call("attn_workspace", self._rows(q), _slab(k, self._dt, self._dev, "DraftTree"),
                          _slab(v, self._dt, self._dev, "DraftTree"), self._desc)

    def verify(self, logits, tokens, accept, sample, draft=None, temperature=1.0, out=None, stream=None):
        """Which nodes stay, and the next token: (path int32 [n_tree, T], n_path int32 [n_tree], token int32 [n_tree]).
        logits (n_tree, T, V): the target's behind each node; tokens int32 [n_tree, T]; accept F32 [n_tree, T] and sample
        F32 [n_tree]: uniform random numbers; draft (n_tree, T, V): the distributions that the nodes' children were drawn
        from, None: fixed choices; temperature 0: greedy.  out: the three results' tensors."""
        if stream is not None:
            with self._on(stream):
                return self.verify(logits, tokens, accept, sample, draft, temperature, out)
        f32 = self._torch.float32
        if sample.dtype is not f32:
            raise MM3FAError(ERR_TYPE, "DraftTree: sample")
        if out is None:
            n, T = self.n_tree, self.max_nodes
            made = self._torch.empty(n * (T + 2), dtype=self._int32, device=self.device)
            out = made[:n * T].view(n, T), made[n * T:n * T + n], made[n * T + n:]
        path, n_path, token = out
        self._run("verify", self._rows_of_nodes(logits, "logits"), None if draft is None else self._rows_of_nodes(draft, "draft"),
                  self._desc, self._each_node(tokens, self._int32, "tokens"), self._each_node(accept, f32, "accept"),
                  self._ints(sample.view(self._int32), self.n_tree, "sample"), temperature,
                  self._each_node(path, self._int32, "path"), self._ints(n_path, self.n_tree, "n_path"),
                  self._ints(token, self.n_tree, "token"), self._stream())
        return out

    def commit(self, layers, path, n_path, kv_len, kv_len_out=None, stream=None):
        """Moves the rows of the nodes on each path behind the cached tokens, in all of `layers` (CacheLayers), and returns
        the new lengths (in kv_len_out where it is given; it may not be kv_len)."""
        if stream is not None:
            with self._on(stream):
                return self.commit(layers, path, n_path, kv_len, kv_len_out)
        if layers.device != self.device:
            raise self._elsewhere(layers)
        if kv_len_out is None:
            kv_len_out = self._torch.empty_like(kv_len)
        n = layers.n_seq
        self._run("commit", *layers._desc, layers.n_layers, self._each_node(path, self._int32, "path"),
                  self._ints(n_path, self.n_tree, "n_path"), self.max_nodes, self.n_tree, self._ints(kv_len, n, "kv_len"),
                  self._ints(kv_len_out, n, "kv_len_out"), self._stream())
        return kv_len_out
