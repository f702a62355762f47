"""The 8-bit paged KV cache (the mm3fa_kv8_* entry points of include/mm3fa.h) on torch tensors.

    cache = mm3fa.Kv8Cache.allocate(n_layers=36, n_pages=512, n_head_kv=8, page_tokens=64, head_dim=128)
    cache.reserve(table, refs, kv_len + 1)                        # pages for the step's rows
    cache.append(layer, k_new, v_new, table, start=kv_len)        # store them as int8 codes
    out = cache.attend(layer, q, table, kv_len + 1, scale)        # attention over the pages
    cache.fork(src, dst, table, kv_len, refs, table2, kv_len2, refs2)   # sequences from others
    cache.compact(table, refs, table2, refs2)                     # live pages to the front

Every call enqueues on torch's current stream (or `stream`) of the cache's device and raises MM3FAError
where the C ABI rejects it; nothing synchronises except `check`.  table is int32 [N, max_pages], kv_len,
q_len, start and n int32 [N], refs int32 [n_pages], all on the cache's device.
"""
from __future__ import annotations

import ctypes
import struct

from . import ERR_SHAPE, ERR_STRIDE, ERR_TYPE, MM3FAError, lib
from .on_device import _PACK_TENSOR, OnDevice  # noqa: F401

FORK_DEEP = 1  # MM3FA_KV8_FORK_DEEP

_CACHE = struct.Struct("@6i4P")                 # struct mm3fa_kv8
_PACK_TABLE = struct.Struct("@Pq2i").pack       # struct mm3fa_kv8_table

_fns = None


def _calls():
    """The library's entry points with their argument types (structs go in as packed bytes)."""
    global _fns
    if _fns is None:
        L, vp, i, sz, f = lib(), ctypes.c_void_p, ctypes.c_int, ctypes.c_size_t, ctypes.c_float
        sigs = {
            "append": (i, [vp, i, vp, vp, vp, vp, vp, vp]),
            "read": (i, [vp, i, vp, vp, vp, vp, vp, vp]),
            "attn_workspace": (sz, [vp, vp, vp]),
            "attn": (i, [vp, i, vp, vp, vp, vp, f, f, i, vp, vp, sz, vp]),
            "pages_workspace": (sz, [vp, i]),
            "reserve": (i, [vp, vp, vp, vp, vp, sz, vp]),
            "fork": (i, [vp, vp, vp, vp, vp, vp, i, ctypes.c_uint32, vp, vp, vp, vp, sz, vp]),
            "compact": (i, [vp, vp, vp, vp, vp, vp, sz, vp]),
        }
        fns = {}
        for name, (res, args) in sigs.items():
            fn = getattr(L, "mm3fa_kv8_" + name)
            fn.restype, fn.argtypes = res, args
            fns[name] = fn
        fns["capture_id"] = fn = L.mm3fa_capture_id
        fn.restype, fn.argtypes = ctypes.c_uint64, [vp]
        _fns = fns
    return _fns


class Kv8Cache(OnDevice):
    """int8 pages [n_layers, n_pages, n_head_kv, page_tokens, head_dim] of K and V and their F32 scales
    [n_layers, n_pages, n_head_kv]; the tensors stay the caller's."""

    def __init__(self, k, v, k_scale, v_scale):
        import torch

        if k.dim() != 5 or k.shape != v.shape or k_scale.shape != k.shape[:3] or v_scale.shape != k.shape[:3]:
            raise MM3FAError(ERR_SHAPE, "Kv8Cache")
        if k.dtype != torch.int8 or v.dtype != torch.int8 or k_scale.dtype != torch.float32 or v_scale.dtype != torch.float32:
            raise MM3FAError(ERR_TYPE, "Kv8Cache")
        if not all(t.is_contiguous() for t in (k, v, k_scale, v_scale)):
            raise MM3FAError(ERR_STRIDE, "Kv8Cache")
        if not all(t.device == k.device for t in (v, k_scale, v_scale)):
            raise ValueError("Kv8Cache: k, v and their scales have to be on one device")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.n_layers, self.n_pages, self.n_head_kv, self.page_tokens, self.head_dim = k.shape
        self._desc = _CACHE.pack(self.head_dim, self.page_tokens, self.n_head_kv, self.n_pages, self.n_layers, 0,
                                 k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr())
        self._on_device_of(k)

    @classmethod
    def allocate(cls, n_layers: int, n_pages: int, n_head_kv: int, page_tokens: int, head_dim: int, device="cuda"):
        """A cache of zeroed pages."""
        import torch

        shape = (n_layers, n_pages, n_head_kv, page_tokens, head_dim)
        codes = [torch.zeros(shape, dtype=torch.int8, device=device) for _ in range(2)]
        scales = [torch.zeros(shape[:3], dtype=torch.float32, device=device) for _ in range(2)]
        return cls(codes[0], codes[1], scales[0], scales[1])

    _prefix = "mm3fa_kv8_"

    def _calls(self):
        return _calls()

    # ------------------------------------------------------------ descriptors

    def _table(self, t):
        if t.dim() != 2:
            raise MM3FAError(ERR_SHAPE, "Kv8Cache: table")
        if t.dtype is not self._int32:
            raise MM3FAError(ERR_TYPE, "Kv8Cache: table")
        if t.get_device() != self._dev:
            raise self._elsewhere(t)
        n, pages = t.shape
        stride, one = t.stride()
        if one != 1 and pages > 1:
            raise MM3FAError(ERR_STRIDE, "Kv8Cache: table")
        return _PACK_TABLE(t.data_ptr(), stride if n > 1 else pages, pages, n)

    # ------------------------------------------------------------ operators

    def append(self, layer, k_new, v_new, table, start, n_new=None, stream=None):
        """Stores the rows k_new, v_new (N, n_head_kv, T, D), the first n_new[s] (default: T) of sequence s, behind
        its first start[s] tokens.  The pages' scales grow where the rows need it."""
        if stream is not None:
            with self._on(stream):
                return self.append(layer, k_new, v_new, table, start, n_new)
        n = table.shape[0]
        self._run("append", self._desc, layer, self._rows(k_new), self._rows(v_new), self._table(table),
                   self._ints(start, n, "start"), None if n_new is None else self._ints(n_new, n, "n_new"),
                   self._stream())

    def read(self, layer, k_out, v_out, table, start, n=None, stream=None):
        """Values of tokens start[s] .. start[s] + n[s] (default: T) of each sequence into the first rows of
        k_out, v_out (N, n_head_kv, T, D)."""
        if stream is not None:
            with self._on(stream):
                return self.read(layer, k_out, v_out, table, start, n)
        ns = table.shape[0]
        self._run("read", self._desc, layer, self._table(table), self._ints(start, ns, "start"),
                   None if n is None else self._ints(n, ns, "n"), self._rows(k_out), self._rows(v_out),
                   self._stream())

    def attend(self, layer, q, table, kv_len, scale, out=None, q_len=None, causal=True, logit_softcap=0.0, ws=None,
               stream=None):
        """softmax(scale * q k^T) v of the queries q (N, n_head, n_q, D) over the first kv_len[s] tokens of each
        sequence; causal: the rows are the last tokens.  out: (N, n_q, n_head, D), F32 or q's type; made in
        q's type when not given, with zeros in the rows behind q_len.  ws: a uint8 tensor, its
        first 64 KiB zero, instead of the cache's own workspace of the stream; it serves one stream at a time.  (Calls in a
        capture that torch.cuda.graph has not begun need one: their graph has no memory of its own.)"""
        if stream is not None:  # what is allocated here belongs to that stream too
            with self._on(stream):
                return self.attend(layer, q, table, kv_len, scale, out, q_len, causal, logit_softcap, ws)
        n = table.shape[0]
        qd, td, st = self._rows(q), self._table(table), self._stream()
        if out is None:
            make = self._torch.empty if q_len is None else self._torch.zeros
            out = make((q.shape[0], q.shape[2], q.shape[1], q.shape[3]), dtype=q.dtype, device=q.device)
        if ws is None:
            shape = (q.shape[2], q.shape[1], n, table.shape[1])
            need = self._need.get(shape)
            if need is None:
                need = self._need[shape] = self._call("attn_workspace", self._desc, qd, td)
            ptr, cap = self._workspace(("attn", st), need)
        else:
            ptr, cap = self._given(ws)
        self._run("attn", self._desc, layer, qd, td, self._ints(kv_len, n, "kv_len"),
                   None if q_len is None else self._ints(q_len, n, "q_len"), scale, logit_softcap, 1 if causal else 0,
                   self._rows(out), ptr, cap, st)
        return out

    def attend_workspace(self, q, table) -> int:
        """Bytes of the workspace that `attend` needs for these operands."""
        return self._call("attn_workspace", self._desc, self._rows(q), self._table(table))

    def _pages_ws(self, n_seq, stream, ws=None):
        if ws is not None:
            return self._given(ws)
        need = self._need.get(n_seq)
        if need is None:
            need = self._need[n_seq] = self._call("pages_workspace", self._desc, n_seq)
        return self._workspace(("pages", stream), need)

    def pages_workspace(self, n_seq) -> int:
        """Bytes of the workspace that `reserve`, `fork`, `free` and `compact` need for n_seq sequences."""
        return self._call("pages_workspace", self._desc, n_seq)

    def reserve(self, table, refs, n_tok, stream=None, ws=None):
        """Gives each sequence's row of `table` the pages for n_tok[s] tokens (in place).  ws: as for `attend`."""
        if stream is not None:
            with self._on(stream):
                return self.reserve(table, refs, n_tok, ws=ws)
        st, n = self._stream(), table.shape[0]
        self._run("reserve", self._desc, self._table(table), self._ints(refs, self.n_pages, "refs"),
                   self._ints(n_tok, n, "n_tok"), *self._pages_ws(n, st, ws), st)

    def fork(self, src, dst, table, kv_len, refs, table_out, kv_len_out, refs_out, deep=False, stream=None, ws=None):
        """Sequence dst[i] becomes a copy of sequence src[i] (-1, or src None: empty); full pages are shared unless
        `deep`.  The results go to the *_out tensors, which may not overlap the others.  ws: as for `attend`."""
        if stream is not None:
            with self._on(stream):
                return self.fork(src, dst, table, kv_len, refs, table_out, kv_len_out, refs_out, deep, ws=ws)
        st, n = self._stream(), table.shape[0]
        pairs = dst.shape[0]
        self._run("fork", self._desc, self._table(table), self._ints(kv_len, n, "kv_len"),
                   self._ints(refs, self.n_pages, "refs"), None if src is None else self._ints(src, pairs, "src"),
                   self._ints(dst, pairs, "dst"), pairs, FORK_DEEP if deep else 0, self._table(table_out),
                   self._ints(kv_len_out, n, "kv_len_out"), self._ints(refs_out, self.n_pages, "refs_out"),
                   *self._pages_ws(n, st, ws), st)

    def free(self, seqs, table, kv_len, refs, table_out, kv_len_out, refs_out, stream=None, ws=None):
        """Empties the sequences `seqs` (int32 [n]): `fork` from nothing."""
        self.fork(None, seqs, table, kv_len, refs, table_out, kv_len_out, refs_out, stream=stream, ws=ws)

    def compact(self, table, refs, table_out, refs_out, stream=None, ws=None):
        """Moves the live pages to the front of the pool; the results go to the *_out tensors.  ws: as for `attend`."""
        if stream is not None:
            with self._on(stream):
                return self.compact(table, refs, table_out, refs_out, ws=ws)
        st, n = self._stream(), table.shape[0]
        self._run("compact", self._desc, self._table(table), self._ints(refs, self.n_pages, "refs"),
                   self._table(table_out), self._ints(refs_out, self.n_pages, "refs_out"), *self._pages_ws(n, st, ws), st)
