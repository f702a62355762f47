"""Calls of the 8-bit paged cache at the edges of what its header promises, on the GPU: against the 64-bit references of
tests/kv8_ref.py, with the helpers of tests/test_kv8_gpu.py."""
import pytest
import torch

import kv8_ref as R
from test_kv8_gpu import DTYPES, many

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
