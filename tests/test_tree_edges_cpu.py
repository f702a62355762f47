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


@no_gpu
def test_attend_refuses_results_in_the_queries_memory():
    """A result's row in memory of a query's, which another CTA may still have to read; rows between one another's are fine."""
    N, H, T, D = 2, 4, 5, 64
    t, k, n, ws = mm3fa.DraftTree(ints(1, T)), torch.zeros(N, 2, 30, D), ints(N), torch.zeros(1 << 24, dtype=torch.uint8)
    a = lambda q, out: status(t.attend, q, k, k, n, 0.1, out=out, ws=ws)
    mem = torch.zeros(8 * N * T * H * D)
    rows = lambda at, sn, st, sh: mem.as_strided((N, T, H, D), (sn, st, sh, 1), at)
    whole = (T * H * D, H * D, D)
    size = N * T * H * D
    q = rows(size, *whole).transpose(1, 2)
    for at, want in ((0, mm3fa.ERR_DEVICE), (2 * size, mm3fa.ERR_DEVICE), (size, mm3fa.ERR_UNSUPPORTED), (1, mm3fa.ERR_UNSUPPORTED),
                     (2 * size - 1, mm3fa.ERR_UNSUPPORTED), (size + D, mm3fa.ERR_UNSUPPORTED)):
        assert a(q, rows(at, *whole)) == want, at
    # queries and results in turn in one buffer: by rows, by nodes, by sequences
    for strides, offs in (((2 * T * H * D, 2 * H * D, 2 * D), D), ((2 * T * H * D, 2 * H * D, D), H * D), ((2 * T * H * D, H * D, D), T * H * D)):
        q = rows(0, *strides).transpose(1, 2)
        assert a(q, rows(offs, *strides)) == mm3fa.ERR_DEVICE
        for off in (0, offs - 1, offs + 1):
            assert a(q, rows(off, *strides)) == mm3fa.ERR_UNSUPPORTED, (strides, off)
    # a 16-bit query's F32 result is twice as wide
    half = mem.half()
    q = half.as_strided((N, T, H, D), (4 * T * H * D, 4 * H * D, 4 * D, 1)).transpose(1, 2)
    f32 = lambda at: half.view(torch.float32).as_strided((N, T, H, D), (2 * T * H * D, 2 * H * D, 2 * D, 1), at)
    assert a(q, f32(D // 2)) == mm3fa.ERR_DEVICE and a(q, f32(D)) == mm3fa.ERR_DEVICE
    assert a(q, f32(0)) == mm3fa.ERR_UNSUPPORTED and a(q, f32(D // 2 - 1)) == mm3fa.ERR_UNSUPPORTED and a(q, f32(D + 1)) == mm3fa.ERR_UNSUPPORTED
    # one query for all heads or nodes
    q = mem[:D].expand(N, H, T, D)
    assert a(q, rows(D, *whole)) == mm3fa.ERR_DEVICE and a(q, rows(D - 1, *whole)) == mm3fa.ERR_UNSUPPORTED
    q = rows(3 * D, 0, 0, 0).transpose(1, 2)
    assert a(q, rows(0, *whole)) == mm3fa.ERR_UNSUPPORTED
