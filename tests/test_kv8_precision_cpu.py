"""The bound of tests/kv8_precision.py holds for 64-bit results and for q and weights of 22 bits, and for none with one of
the two rounded to 11 or 8."""
import pytest
import torch

import kv8_precision as E
import kv8_ref as R


def pair(x):
    """A number as the sum of two F16 numbers: 22 bits."""
    hi = x.to(torch.float16).double()
    return hi + (x.double() - hi).to(torch.float16).double()


@pytest.mark.parametrize("lens,n_q", [([64, 90], 1), ([300, 500], 1), ([300, 220], 16), ([3001, 9999], 1), ([700, 1500], 8)])
def test_the_bound_tells_22_bits_from_11(lens, n_q):
    st = R.State(lens, 2, 128, 64, seed=27)
    q = st.randn(2, 8, n_q, 128)
    assert E.worst(st, q, E.simulate(st, q)) < 1e-6
    assert E.worst(st, q, E.simulate(st, pair(q))) < 0.2
    for t in (torch.float16, torch.bfloat16):
        assert E.worst(st, q, E.simulate(st, q, q_type=t)) > 2
        assert E.worst(st, q, E.simulate(st, q, w_type=t)) > 2
