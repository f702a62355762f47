"""What the operators of tree decoding refuse where a call would give results that depend on timing, on host tensors."""
import pytest
import torch

import mm3fa
from mm3fa import tree as T_
from test_tree_cpu import ints, no_gpu, status


@no_gpu
def test_commit_refuses_lengths_in_memory_that_it_reads():
    """The new lengths replace nothing that another warp or a later launch still reads: kv_len, the paths, their counts."""
    N, T = 2, 5
    t, k = mm3fa.DraftTree(ints(N, T)), torch.zeros(3, N, 2, 30, 64, dtype=torch.float16)
    mem = ints(100)
    path, n_path, n, m = mem[:N * T].view(N, T), mem[20:20 + N], mem[40:40 + N], mem[60:60 + N]
    a = lambda out: status(t.commit, mm3fa.CacheLayers(k, k), path, n_path, n, kv_len_out=out)
    assert a(m) == mm3fa.ERR_DEVICE
    for out in (n, n_path, mem[:N], mem[4:4 + N], mem[N * T - N:N * T]):
        assert a(out) == mm3fa.ERR_UNSUPPORTED
    # its last or its first entry is one of theirs
    for at, size in ((0, N * T), (20, N), (40, N)):
        for start, want in ((at - N, mm3fa.ERR_DEVICE), (at - 1, mm3fa.ERR_UNSUPPORTED), (at + size - 1, mm3fa.ERR_UNSUPPORTED), (at + size, mm3fa.ERR_DEVICE)):
            if start >= 0:
                assert a(mem[start:start + N]) == want, (at, start)
