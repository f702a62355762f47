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

from . import ERR_SHAPE, ERR_STRIDE, ERR_TYPE, OK, MM3FAError, lib, workspace_status
from .ggml import GGML_TYPE_BF16, GGML_TYPE_F16, GGML_TYPE_F32

FORK_DEEP = 1  # MM3FA_KV8_FORK_DEEP

_CACHE = struct.Struct("@6i4P")                 # struct mm3fa_kv8
_PACK_TABLE = struct.Struct("@Pq2i").pack       # struct mm3fa_kv8_table
_PACK_TENSOR = struct.Struct("@2i4q4QP").pack   # struct mm3fa_tensor

_ZEROED = 1 << 16  # bytes of a workspace that have to be zero before its first use
_ALSO = slice(16, 24)  # of a workspace: address of a second status word

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


_STATUS_SLOTS = 1 << 16
_status_words = {}  # device -> [int32 [_STATUS_SLOTS, 4], slots given out]


def _status_memory(device):
    """Status words for calls of graphs, of which a graph keeps the address: never freed, and none given out twice (but in
    turn when all have been)."""
    import torch

    if device not in _status_words:
        _status_words[device] = [torch.zeros(_STATUS_SLOTS, 4, dtype=torch.int32, device=device), 0]
    return _status_words[device]


def _types():
    import torch

    return {torch.float32: (GGML_TYPE_F32, 4), torch.float16: (GGML_TYPE_F16, 2), torch.bfloat16: (GGML_TYPE_BF16, 2)}


class Kv8Cache:
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
        self.device = k.device
        self.n_layers, self.n_pages, self.n_head_kv, self.page_tokens, self.head_dim = k.shape
        self._desc = _CACHE.pack(self.head_dim, self.page_tokens, self.n_head_kv, self.n_pages, self.n_layers, 0,
                                 k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr())
        self._torch, self._int32 = torch, torch.int32
        self._dt = _types()
        self._dev = k.get_device()  # -1: host tensors, on which the C ABI's checks run but no kernel does
        self._fns = None
        self._ws = {}    # (operation, stream) -> address and bytes of a zero-filled workspace
        self._kept = []  # these, outgrown ones too: their status has not been read
        self._need = {}  # workspace bytes by shape
        self._capture = None  # the last capture, and its workspaces by (operation, stream)
        self._is_capturing, self._current_device = torch._C._cuda_isCurrentStreamCapturing, torch._C._cuda_getDevice
        self._found = {}  # (operation, stream), or None: the status of calls of graphs
        self._status = None if self._dev < 0 else _status_memory(self.device)

    @classmethod
    def allocate(cls, n_layers: int, n_pages: int, n_head_kv: int, page_tokens: int, head_dim: int, device="cuda"):
        """A cache of zeroed pages."""
        import torch

        shape = (n_layers, n_pages, n_head_kv, page_tokens, head_dim)
        codes = [torch.zeros(shape, dtype=torch.int8, device=device) for _ in range(2)]
        scales = [torch.zeros(shape[:3], dtype=torch.float32, device=device) for _ in range(2)]
        return cls(codes[0], codes[1], scales[0], scales[1])

    # ------------------------------------------------------------ descriptors

    def _elsewhere(self, t):
        return ValueError(f"Kv8Cache: a tensor on {t.device}, the cache is on {self.device}")

    def _rows(self, t):
        """mm3fa_tensor [D, rows, heads, seqs] of a torch tensor (seqs, heads, rows, D)."""
        if t.dim() != 4:
            raise MM3FAError(ERR_SHAPE, "Kv8Cache: rows of 4 dimensions are wanted")
        ty = self._dt.get(t.dtype)
        if ty is None:
            raise MM3FAError(ERR_TYPE, "Kv8Cache")
        if t.get_device() != self._dev:
            raise self._elsewhere(t)
        a, b, c, d = t.shape
        sa, sb, sc, sd = t.stride()
        if sd != 1 and d > 1:
            raise MM3FAError(ERR_STRIDE, "Kv8Cache: the head dimension has to be contiguous")
        ty, e = ty
        return _PACK_TENSOR(ty, 0, d, c, b, a, e, sc * e, sb * e, sa * e, t.data_ptr())

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

    def _ints(self, t, n, what):
        """Address of an int32 tensor of n entries."""
        if t.dtype is not self._int32:
            raise MM3FAError(ERR_TYPE, "Kv8Cache: " + what)
        if t.get_device() != self._dev:
            raise self._elsewhere(t)
        if t.dim() != 1 or t.shape[0] != n:
            raise MM3FAError(ERR_SHAPE, "Kv8Cache: " + what)
        if n > 1 and t.stride(0) != 1:
            raise MM3FAError(ERR_STRIDE, "Kv8Cache: " + what)
        return t.data_ptr()

    def _stream(self):
        return 0 if self._dev < 0 else self._torch._C._cuda_getCurrentRawStream(self._dev)

    def _on(self, stream):
        """A context in which `stream` is the current one."""
        if stream.device_index != self._dev:
            raise ValueError(f"Kv8Cache: a stream of device {stream.device_index}, the cache is on {self.device}")
        return self._torch.cuda.stream(stream)

    def _call(self, name, *args):
        """A library call with the cache's device current; its result."""
        fn = (self._fns or self._bind())[name]
        if self._dev < 0 or self._torch._C._cuda_getDevice() == self._dev:
            return fn(*args)
        with self._torch.cuda.device(self.device):
            return fn(*args)

    def _bind(self):
        self._fns = _calls()
        return self._fns

    def _run(self, name, *args):
        st = self._call(name, *args)
        if st:
            raise MM3FAError(st, "mm3fa_kv8_" + name)

    def _workspace(self, key, nbytes):
        """(address, bytes) of the workspace of an operation on a stream, zero-filled as far as it has to be when it is made."""
        # the current stream is key's where the current device is the cache's
        if self._dev >= 0 and (self._is_capturing() or self._current_device() != self._dev):
            capture = self._call("capture_id", key[1])
            if capture:
                return self._workspace_of_graph(capture, key, nbytes)
        if self._capture:
            self._capture = None
        buf = self._ws.get(key)
        if buf is not None and buf[1] >= nbytes:
            return buf
        if nbytes > 0:
            made = self._made(nbytes)
            self._ws[key] = at = made.data_ptr(), made.numel()
            self._kept.append((key, made))
            return at
        return None, 0

    def _made(self, nbytes):
        made = self._torch.empty(max(nbytes, _ZEROED), dtype=self._torch.uint8, device=self.device)
        made[:_ZEROED].zero_()
        return made

    def _workspace_of_graph(self, capture, key, nbytes):
        """A workspace that a graph zeroes when it is replayed: one for all calls of an operation that a stream of the
        capture makes, shared with nothing else.  It lives in the graph's memory, like all that is allocated in a
        capture; this class lets it go at its next call elsewhere (one that the capture makes later is zeroed in turn).
        What the calls find goes to a status word of the stream where it has a workspace, else to one of the cache."""
        if self._capture is None or self._capture[0] != capture:
            self._capture = capture, {}
        made = self._capture[1].get(key)
        if made is None or made.numel() < nbytes:
            if nbytes <= 0:
                return None, 0
            made = self._capture[1][key] = self._made(nbytes)
            made[_ALSO].view(self._torch.int64).fill_(self._status_word(key if key in self._ws else None).data_ptr())
        return made.data_ptr(), made.numel()

    def _status_word(self, key):
        word = self._found.get(key)
        if word is None:
            words, n = self._status
            self._status[1] = n + 1
            word = self._found[key] = words[n % _STATUS_SLOTS]
        return word

    def _given(self, ws):
        """(address, bytes) of a caller's workspace."""
        if ws.get_device() != self._dev:
            raise self._elsewhere(ws)
        if not ws.is_contiguous():
            raise MM3FAError(ERR_STRIDE, "Kv8Cache: workspace")
        return ws.data_ptr(), ws.numel() * ws.element_size()

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

    def check(self, stream=None, captured=False, ws=None):
        """Synchronises the stream and raises MM3FAError where a page operation on it found too few free pages
        (ERR_PAGES) or a bounded device wait of an attention expired (ERR_TIMEOUT).  Calls that a graph replays are among
        them where an earlier call on the stream of the capture had made its workspace; captured=True: those of all
        graphs (wait for the streams that replay them first).  ws: a workspace that calls were given."""
        if stream is not None:
            with self._on(stream):
                return self.check(captured=captured, ws=ws)
        st = self._stream()
        bufs = [buf for key, buf in self._kept if key[1] == st]  # outgrown ones too
        bufs += [word for key, word in self._found.items() if captured or (key and key[1] == st)]
        bufs += [ws] if ws is not None else []
        for buf in bufs:
            status, _ = workspace_status(buf.data_ptr(), st)
            if status != OK:
                raise MM3FAError(status, "Kv8Cache")
