"""Calls of the 8-bit paged cache at the edges of what its header promises, on the GPU: against the 64-bit references of
tests/kv8_ref.py, with the helpers of tests/test_kv8_gpu.py."""
import pytest
import torch

import kv8_ref as R
import mm3fa
from test_kv8_gpu import DTYPES, many, run_attend

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("softcap", [0.0, 5.0])
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("D,G,n_q,n0", [(64, 2, 1, 1), (128, 2, 4, 1), (64, 2, 70, 30), (128, 2, 70, 30), (64, 1, 200, 199),
                                        (128, 1, 300, 200), (128, 2, 200, 199)])
def test_attend_nan_in_a_row_that_sees_no_key(cuda_device, D, G, n_q, n0, dtype, softcap):
    """A row that sees no key is zeros though its q holds a NaN or an infinity: the first rows of a causal call with
    more rows than keys, beside rows that see a few or a whole tile of them, and those of a sequence all of whose pages are
    missing.  A row of NaN that sees a key is NaN; the rest is what it is without them."""
    dt = DTYPES[dtype]
    st = many(R.State([n0, 300], 2, D, 64, seed=24, device=cuda_device), G * n_q)
    st.table[1] = -1
    q = st.randn(st.N, 2 * G, n_q, D).to(dt)
    cap = dict(logit_softcap=softcap)
    want = st.cache().attend(0, q, st.table, st.len, 0.125, **cap)
    assert (want[1] == 0).all()
    hidden = max(0, n_q - n0)  # rows of sequence 0 that see no key
    assert (want[0, :hidden] == 0).all()
    for bad in (float("nan"), float("inf")):
        q2 = q.clone()
        q2[0, 1, :, 3] = bad
        q2[1, 0, :, 5] = bad
        got = st.cache().attend(0, q2, st.table, st.len, 0.125, **cap)
        assert (got[1] == 0).all()
        assert (got[0, :hidden] == 0).all()
        assert got[0, hidden:, 1].isnan().all()
        got[0, hidden:, 1] = want[0, hidden:, 1]
        assert torch.equal(got, want)


def test_wait_limit_starts_after_the_previous_kernel(cuda_device, tmp_path):
    """The bounded waits of the many-row kernel count from its own start.  It is launched behind a peer wait, which lets its
    successor launch at once and then runs to its own limit: that time is not the attention's.  In a process of its own,
    with a limit of 1 ms."""
    import os
    import subprocess
    import sys

    here = os.path.dirname(os.path.abspath(__file__))
    code = f"""
import ctypes, sys
sys.path[:0] = [{here!r}, {os.path.join(os.path.dirname(here), "minimaxmusic.cpp_b200")!r}]
import torch
import kv8_ref as R
import mm3fa
import mm3fa
from mm3fa import ggml
dev = torch.device("cuda", 0)
st = R.State([4000] * 8, 4, 128, 64, seed=31, device=dev)
c, q = st.cache(), st.randn(8, 8, 512, 128)
want = c.attend(0, q, st.table, st.len, 0.1, logit_softcap=5.0).clone()
c.check()
recv, epochs, ws = (torch.zeros(n, dtype=torch.uint8, device=dev) for n in (1 << 20, 256, 1 << 16))
res = torch.zeros(1, 1, 4, 128, device=dev)
peers = mm3fa.Peers()
peers.n_ranks, peers.rank, peers.recv_slot_bytes = 2, 0, 1 << 20
peers.recv[0] = peers.recv[1] = recv.data_ptr()
s = torch.cuda.current_stream().cuda_stream
for _ in range(20):
    out = torch.zeros_like(want)
    mm3fa.peer_wait(peers, 0, epochs.data_ptr(), ggml.make(ggml.GGML_TYPE_F32, [128, 4, 1, 1], res.data_ptr()), ws.data_ptr(), s)
    c.attend(0, q, st.table, st.len, 0.1, out=out, logit_softcap=5.0)
    c.check()
    assert torch.equal(out, want)
    assert mm3fa.workspace_status(ws.data_ptr(), s)[0] == mm3fa.ERR_TIMEOUT  # the peer's words never come
print("done")
"""
    r = subprocess.run([sys.executable, "-c", code], env={**os.environ, "MM3FA_WAIT_TIMEOUT_MS": "1"}, capture_output=True,
                       text=True, timeout=300)
    assert r.returncode == 0 and "done" in r.stdout, r.stdout + r.stderr


# ---------------------------------------------------------------- graphs

def small_cache(dev, n_pages=6, n_free=0):
    """A cache of n_pages pages of which n_free are free, and a table of one sequence without any."""
    c = mm3fa.Kv8Cache.allocate(3, n_pages, 2, 16, 64, dev)
    refs = torch.ones(n_pages, dtype=torch.int32, device=dev)
    refs[:n_free] = 0
    return c, refs, torch.full((1, 4), -1, dtype=torch.int32, device=dev)


def captured(fn, stream=None):
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        fn()
    return g


def test_captured_calls_share_a_workspace_that_goes_with_the_graph(cuda_device):
    """36 attentions of one capture hold one workspace, and none when the graph is gone."""
    st = R.State([500, 1200], 4, 128, 64, seed=32, device=cuda_device)
    c, q = st.cache(), st.randn(2, 16, 1, 128)
    outs = torch.zeros(36, 2, 1, 16, 128, device=cuda_device)
    want = c.attend(0, q, st.table, st.len, 0.1).clone()
    need = c.attend_workspace(q, st.table)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    g = captured(lambda: [c.attend(0, q, st.table, st.len, 0.1, out=o) for o in outs])
    assert torch.cuda.memory_allocated() - before <= 2 * need
    for _ in range(2):
        outs.zero_()
        g.replay()
        assert all(torch.equal(o, want) for o in outs)
    del g
    c.attend(0, q, st.table, st.len, 0.1)  # lets go of the capture
    torch.cuda.synchronize()
    assert torch.cuda.memory_allocated() == before


def test_captured_calls_that_outgrow_their_workspace(cuda_device):
    """Calls of growing and of alternating shapes in one capture, with other allocations between them."""
    sts = [R.State([9000, 700], 8, D, 64, seed=D, device=cuda_device) for D in (64, 128)]
    shapes = [(st, n_q) for n_q in (1, 40, 2) for st in sts]
    qs = [st.randn(2, 16, n_q, st.D) for st, n_q in shapes]
    caches = [st.cache() for st in sts]
    want = [caches[i % 2].attend(0, q, st.table, st.len, 0.1).clone() for i, ((st, _), q) in enumerate(zip(shapes, qs))]
    got = []

    def calls():
        for i, ((st, _), q) in enumerate(zip(shapes, qs)):
            got.append(caches[i % 2].attend(0, q, st.table, st.len, 0.1))
            got.append(torch.full((1 << 20,), 255, dtype=torch.uint8, device=cuda_device))

    g = captured(calls)
    for _ in range(3):
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got[::2], want))


def test_a_replayed_call_without_pages_is_reported(cuda_device):
    """check(captured=True) raises for it, though replays that found pages came after it, and only once; the default
    reads what streams of the program's own have found."""
    c, refs, table = small_cache(cuda_device)
    n_tok = torch.ones(1, dtype=torch.int32, device=cuda_device)
    g = captured(lambda: c.reserve(table, refs, n_tok))
    c.check(captured=True)  # nothing has run
    g.replay()
    refs[3] = 0
    g.replay()
    assert int(table[0, 0]) == 3
    torch.cuda.synchronize()
    with pytest.raises(mm3fa.MM3FAError) as e:
        c.check(captured=True)
    assert e.value.status == mm3fa.ERR_PAGES
    c.check(captured=True)
    table.fill_(-1)
    g.replay()  # no page again
    torch.cuda.synchronize()
    with pytest.raises(mm3fa.MM3FAError):
        c.check(captured=True)
    other, _, _ = small_cache(cuda_device)
    g.replay()
    torch.cuda.synchronize()
    other.check(captured=True)  # another cache's status is its own


def test_a_replayed_fork_without_pages_is_reported(cuda_device):
    c, refs, table = small_cache(cuda_device)
    table = torch.tensor([[0, -1], [-1, -1]], dtype=torch.int32, device=cuda_device)
    n = torch.tensor([5, 0], dtype=torch.int32, device=cuda_device)
    pair = [torch.tensor([i], dtype=torch.int32, device=cuda_device) for i in (0, 1)]
    outs = [torch.empty_like(t) for t in (table, n, refs)]
    g = captured(lambda: c.fork(*pair, table, n, refs, *outs))
    g.replay()
    torch.cuda.synchronize()
    with pytest.raises(mm3fa.MM3FAError) as e:
        c.check(captured=True)
    assert e.value.status == mm3fa.ERR_PAGES
    assert torch.equal(outs[0], table)


def test_graphs_of_one_stream_at_the_same_time(cuda_device):
    """Two graphs captured on a stream that has a workspace, replayed on two streams while a third makes eager calls: none
    shares a workspace with another."""
    st = R.State([3000, 5000], 4, 128, 64, seed=33, device=cuda_device)
    c = st.cache()
    qs = [st.randn(2, 16, n_q, 128) for n_q in (1, 3, 2)]
    side = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    with torch.cuda.stream(side[0]):
        want = [c.attend(0, q, st.table, st.len, 0.1).clone() for q in qs]
    torch.cuda.synchronize()
    outs = [[torch.empty_like(w) for _ in range(8)] for w in want]
    graphs = [captured(lambda: [c.attend(0, q, st.table, st.len, 0.1, out=o) for o in os], side[0]) for q, os in zip(qs, outs[:2])]
    for _ in range(20):
        for g, s in zip(graphs, side[1:]):
            with torch.cuda.stream(s):
                g.replay()
        with torch.cuda.stream(side[0]):
            for o in outs[2]:
                c.attend(0, qs[2], st.table, st.len, 0.1, out=o)
    torch.cuda.synchronize()
    for w, os in zip(want, outs):
        assert all(torch.equal(o, w) for o in os)


def test_a_workspace_for_page_operations(cuda_device):
    """reserve, fork, free and compact with a workspace of the caller's, eager and captured; check reads it."""
    c, refs, table = small_cache(cuda_device, n_free=2)
    ws = torch.zeros(c.pages_workspace(1), dtype=torch.uint8, device=cuda_device)
    ws[1 << 16:] = 255
    n_tok = torch.full((1,), 17, dtype=torch.int32, device=cuda_device)
    c.reserve(table, refs, n_tok, ws=ws)
    c.check(ws=ws)
    assert table.tolist() == [[0, 1, -1, -1]]
    outs = [torch.empty_like(t) for t in (table, n_tok, refs)]
    zero = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    c.free(zero, table, n_tok, refs, *outs, ws=ws)
    assert outs[0].tolist() == [[-1] * 4] and outs[2].tolist() == [0, 0, 1, 1, 1, 1]
    t2, r2 = torch.empty_like(table), torch.empty_like(refs)
    c.compact(outs[0], outs[2], t2, r2, ws=ws)
    assert r2.tolist() == [1, 1, 1, 1, 0, 0]
    refs.fill_(1)
    table.fill_(-1)
    torch.cuda.synchronize()
    g = captured(lambda: c.reserve(table, refs, n_tok, ws=ws))
    g.replay()
    torch.cuda.synchronize()
    c.check(captured=True)
    with pytest.raises(mm3fa.MM3FAError) as e:
        c.check(ws=ws)
    assert e.value.status == mm3fa.ERR_PAGES
    c.check(ws=ws)
    for bad in (ws.cpu(), ):
        with pytest.raises(ValueError):
            c.reserve(table, refs, n_tok, ws=bad)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("n_q", [1, 70])
def test_attend_causal_length_beyond_the_table(cuda_device, n_q, dtype):
    """A length beyond the table is the table's, for the causal rows too: the last row sees all of its tokens."""
    st = R.State([128, 64, 10], 2, 64, 64, seed=36, device=cuda_device)
    st.len = torch.tensor([2 ** 31 - 1, -5, 200], dtype=torch.int32, device=cuda_device)
    run_attend(st, 4, n_q, DTYPES[dtype])
