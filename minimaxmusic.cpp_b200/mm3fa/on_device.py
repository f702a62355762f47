"""What classes over torch tensors of one device share: descriptors, calls of the C ABI with that device current, and
zero-filled workspaces, one for each operation and stream, or for each capture."""
from __future__ import annotations

import struct

from . import ERR_SHAPE, ERR_STRIDE, ERR_TYPE, OK, MM3FAError, workspace_status
from .ggml import GGML_TYPE_BF16, GGML_TYPE_F16, GGML_TYPE_F32

_PACK_TENSOR = struct.Struct("@2i4q4QP").pack   # struct mm3fa_tensor

_ZEROED = 1 << 16  # bytes of a workspace that have to be zero before its first use
_ALSO = slice(16, 24)  # of a workspace: address of a second status word

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


class OnDevice:
    """Calls on tensors of one device; subclasses give `_prefix` and `_calls`, the entry points by their names."""

    _prefix = "mm3fa_"

    def _on_device_of(self, t):
        import torch

        self._name = type(self).__name__
        self.device = t.device
        self._torch, self._int32 = torch, torch.int32
        self._dt = _types()
        self._dev = t.get_device()  # -1: host tensors, on which the C ABI's checks run but no kernel does
        self._fns = None
        self._ws = {}    # (operation, stream) -> address and bytes of a zero-filled workspace
        self._kept = []  # these, outgrown ones too: their status has not been read
        self._need = {}  # workspace bytes by shape
        self._capture = None  # the last capture, and its workspaces by (operation, stream)
        self._is_capturing, self._current_device = torch._C._cuda_isCurrentStreamCapturing, torch._C._cuda_getDevice
        self._found = {}  # (operation, stream), or None: the status of calls of graphs
        self._status = None if self._dev < 0 else _status_memory(self.device)

    def _elsewhere(self, t):
        return ValueError(f"{self._name}: a tensor on {t.device}, the others are on {self.device}")

    def _rows(self, t):
        """mm3fa_tensor [D, rows, heads, seqs] of a torch tensor (seqs, heads, rows, D)."""
        if t.dim() != 4:
            raise MM3FAError(ERR_SHAPE, self._name + ": rows of 4 dimensions are wanted")
        ty = self._dt.get(t.dtype)
        if ty is None:
            raise MM3FAError(ERR_TYPE, self._name)
        if t.get_device() != self._dev:
            raise self._elsewhere(t)
        a, b, c, d = t.shape
        sa, sb, sc, sd = t.stride()
        if sd != 1 and d > 1:
            raise MM3FAError(ERR_STRIDE, self._name + ": the head dimension has to be contiguous")
        ty, e = ty
        return _PACK_TENSOR(ty, 0, d, c, b, a, e, sc * e, sb * e, sa * e, t.data_ptr())

    def _ints(self, t, n, what):
        """Address of an int32 tensor of n entries."""
        if t.dtype is not self._int32:
            raise MM3FAError(ERR_TYPE, self._name + ": " + what)
        if t.get_device() != self._dev:
            raise self._elsewhere(t)
        if t.dim() != 1 or t.shape[0] != n:
            raise MM3FAError(ERR_SHAPE, self._name + ": " + what)
        if n > 1 and t.stride(0) != 1:
            raise MM3FAError(ERR_STRIDE, self._name + ": " + what)
        return t.data_ptr()

    def _stream(self):
        return 0 if self._dev < 0 else self._torch._C._cuda_getCurrentRawStream(self._dev)

    def _on(self, stream):
        """A context in which `stream` is the current one."""
        if stream.device_index != self._dev:
            raise ValueError(f"{self._name}: a stream of device {stream.device_index}, the others are on {self.device}")
        return self._torch.cuda.stream(stream)

    def _call(self, name, *args):
        """A library call with that device current; its result."""
        fn = (self._fns or self._bind())[name]
        if self._dev < 0 or self._torch._C._cuda_getDevice() == self._dev:
            return fn(*args)
        with self._torch.cuda.device(self.device):
            return fn(*args)

    def _bind(self):
        self._fns = self._calls()
        return self._fns

    def _run(self, name, *args):
        st = self._call(name, *args)
        if st:
            raise MM3FAError(st, self._prefix + name)

    def _workspace(self, key, nbytes):
        """(address, bytes) of the workspace of an operation on a stream, zero-filled as far as it has to be when it is made."""
        # the current stream is key's where the current device is this one
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
        What the calls find goes to a status word of the stream where it has a workspace, else to one of this object."""
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
            raise MM3FAError(ERR_STRIDE, self._name + ": workspace")
        return ws.data_ptr(), ws.numel() * ws.element_size()

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
                raise MM3FAError(status, self._name)
