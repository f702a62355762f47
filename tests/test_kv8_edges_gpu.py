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
