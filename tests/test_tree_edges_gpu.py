"""Tree decoding on the GPU where its ranges end, against the 64-bit references of tests/tree_ref.py."""
import pytest
import torch

import mm3fa
import tree_ref as R
from test_tree_gpu import Case

pytestmark = pytest.mark.gpu

SIXTEEN = [("f32", "f16"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "bf16"), ("f16", "bf16"), ("bf16", "f16")]


@pytest.mark.parametrize("dtype,cache", SIXTEEN + [("f32", "f32")])
@pytest.mark.parametrize("D", [64, 128])
def test_attend_scales_whose_products_leave_f32(cuda_device, D, dtype, cache):
    """Scales and rows of q so small that a score's factor would be 0, and so large that it would be infinite: the first see
    all keys alike (the mean of the visible V rows), and so do rows of zeros under the second."""
    c = Case(cuda_device, [300, 5, 0], 1, 8, 2, D, 10, dtype, cache, seed=D)
    q = c.q
    for small in (2.0 ** -12, 2.0 ** -60 if dtype != "f16" else 2.0 ** -20):
        c.q = (q.float() * small).to(q.dtype)
        for kw in ({"scale": 0.0}, {"scale": 1e-30}, {"scale": -1e-38}, {"scale": 0.0, "logit_softcap": 2.0}, {"scale": 1e-38, "logit_softcap": 30.0}):
            c.check(**kw)
    c.q = torch.zeros_like(q)
    for kw in ({"scale": 3e38}, {"scale": -3e38}, {"scale": 1e30, "logit_softcap": 1e-20}):
        c.check(**kw)
