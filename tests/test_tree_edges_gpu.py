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


@pytest.mark.parametrize("dtype,cache", [("f32", "f16"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "f32")])
@pytest.mark.parametrize("which", ["k", "v", "kv"])
def test_attend_slabs_of_one_row(cuda_device, which, dtype, cache):
    """n_kv = 1: the row stride is never used, whatever it is (262 bytes are not a multiple of 16, 0 is below a row)."""
    for N, Hkv in ((2, 2), (1, 1), (3, 1), (1, 2)):
        for row in (131, 0):
            c = Case(cuda_device, [i % 2 for i in range(N)], 1, 2 * Hkv, Hkv, 128, 3, dtype, cache, seed=N, rows=1)
            for name in which:
                x = getattr(c, name)
                big = torch.full((N, Hkv, 8, 131), float("nan"), dtype=x.dtype, device=cuda_device)
                view = big.as_strided((N, Hkv, 1, 128), (Hkv * 8 * 131, 8 * 131, row, 1))
                view.copy_(x)
                setattr(c, name, view)
            c.check()
