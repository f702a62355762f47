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
        self.n_layers, self.device, self._sets = len(self.k), self.k[0].device, self.k[0].shape[:1]
        types, dev = _types(), self.k[0].get_device()
        self._desc = [b"".join(_slab(t, types, dev, "CacheLayers") for t in x) for x in (self.k, self.v)]


class DraftTree(OnDevice):
    """Trees of up to 256 drafted tokens: parents int32 [n_tree, T], n_nodes int32 [n_tree] or None (T).  Both are read by every
    call, so that one object serves a program's steps with new trees written over the last ones; it keeps the attention's
    workspace of each stream (up to some 20 MB), which another object would make anew."""

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
        self._each, self._per_node = self._torch.Size((self.n_tree,)), parents.shape
        self._f32 = self._torch.float32
        # results of `verify` are made like these
        self._nodes_like = parents if parents.is_contiguous() else self._torch.empty_like(parents, memory_format=self._torch.contiguous_format)
        self._trees_like = self._torch.empty(self.n_tree, dtype=self._int32, device=self.device)
        counts = 0 if n_nodes is None else self._ints(n_nodes, self.n_tree, "n_nodes")
        self._desc = _PACK_TREE(parents.data_ptr(), parents.stride(0) if self.n_tree > 1 else self.max_nodes, counts,
                                self.max_nodes, self.n_tree)

    def _calls(self):
        return _calls()

    def _flat(self, t, dtype, shape, what):
        """Address of a contiguous tensor of a type and shape."""
        if t.dtype is dtype and t.shape == shape and t.get_device() == self._dev and t.is_contiguous():
            return t.data_ptr()
        if t.dtype is not dtype:
            raise MM3FAError(ERR_TYPE, "DraftTree: " + what)
        if t.get_device() != self._dev:
            raise self._elsewhere(t)
        raise MM3FAError(ERR_SHAPE if t.shape != shape else ERR_STRIDE, "DraftTree: " + what)

    def _rows_of_nodes(self, t, what):
        """mm3fa_tensor [V, T, n_tree, 1] of a tensor (n_tree, T, V)."""
        if t.dim() != 3:
            raise MM3FAError(ERR_SHAPE, "DraftTree: " + what)
        ty = self._dt.get(t.dtype)
        if ty is None:
            raise MM3FAError(ERR_TYPE, "DraftTree: " + what)
        if t.get_device() != self._dev:
            raise self._elsewhere(t)
        n, T, V = t.shape
        sn, st, sv = t.stride()
        if sv != 1 and V > 1:
            raise MM3FAError(ERR_STRIDE, "DraftTree: " + what)
        ty, e = ty
        return _PACK_TENSOR(ty, 0, V, T, n, 1, e, st * e, sn * e, n * sn * e, t.data_ptr())

    def attend(self, q, k, v, kv_len, scale, out=None, logit_softcap=0.0, ws=None, stream=None):
        """softmax(scale * q k^T) v of the queries q (N, n_head, T, D), where node i of a sequence sees the first kv_len[s]
        rows of its slabs k, v (N, n_head_kv, rows, D), and row kv_len[s] + j for itself and its ancestors j.
        out: (N, T, n_head, D), F32 or q's type, not in q's memory; made in q's type when not given, with zeros in the rows of
        nodes that do not count.  ws: a uint8 tensor, its first 64 KiB zero, instead of this object's own workspace of the stream; it serves
        one stream at a time.  (Calls in a capture that torch.cuda.graph has not begun need one.)"""
        if stream is not None:  # what is allocated here belongs to that stream too
            with self._on(stream):
                return self.attend(q, k, v, kv_len, scale, out, logit_softcap, ws)
        qd, st = self._rows(q), self._stream()
        kd, vd = _slab(k, self._dt, self._dev, "DraftTree"), _slab(v, self._dt, self._dev, "DraftTree")
        shape = q.shape
        if out is None:
            make = self._torch.empty if self.n_nodes is None else self._torch.zeros
            out = make((shape[0], shape[2], shape[1], shape[3]), dtype=q.dtype, device=q.device)
        if ws is None:
            key = shape, k.shape, k.dtype
            need = self._need.get(key)
            if need is None:
                need = self._call("attn_workspace", qd, kd, vd, self._desc)
                if need:  # (0: the call is refused, and others of that shape may not be)
                    self._need[key] = need
            ptr, cap = self._workspace(("attn", st), need)
        else:
            ptr, cap = self._given(ws)
        self._run("attn", qd, kd, vd, self._desc, self._flat(kv_len, self._int32, shape[:1], "kv_len"), scale, logit_softcap, self._rows(out),
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
        i32, f32, each, per_node, flat = self._int32, self._f32, self._each, self._per_node, self._flat
        if out is None:
            like = self._torch.empty_like  # (a third of what empty() takes)
            out = like(self._nodes_like), like(self._trees_like), like(self._trees_like)
        path, n_path, token = out
        self._run("verify", self._rows_of_nodes(logits, "logits"), None if draft is None else self._rows_of_nodes(draft, "draft"),
                  self._desc, flat(tokens, i32, per_node, "tokens"), flat(accept, f32, per_node, "accept"),
                  flat(sample, f32, each, "sample"), temperature, flat(path, i32, per_node, "path"),
                  flat(n_path, i32, each, "n_path"), flat(token, i32, each, "token"), self._stream())
        return out

    def commit(self, layers, path, n_path, kv_len, kv_len_out=None, stream=None):
        """Moves the rows of the nodes on each path behind the cached tokens, in all of `layers` (CacheLayers), and returns
        the new lengths (in kv_len_out where it is given; it may not be in the memory of kv_len, path or n_path)."""
        if stream is not None:
            with self._on(stream):
                return self.commit(layers, path, n_path, kv_len, kv_len_out)
        if layers.device != self.device:
            raise self._elsewhere(layers)
        if kv_len_out is None:
            kv_len_out = self._torch.empty_like(kv_len)
        i32, flat, sets = self._int32, self._flat, layers._sets
        self._run("commit", *layers._desc, layers.n_layers, flat(path, i32, self._per_node, "path"),
                  flat(n_path, i32, self._each, "n_path"), self.max_nodes, self.n_tree, flat(kv_len, i32, sets, "kv_len"),
                  flat(kv_len_out, i32, sets, "kv_len_out"), self._stream())
        return kv_len_out
