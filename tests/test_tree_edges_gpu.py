"""Tree decoding on the GPU where its ranges end, against the 64-bit references of tests/tree_ref.py."""
import random

import pytest
import torch

import mm3fa
import tree_ref as R
from test_tree_gpu import Case, check_verify, rising, slabs

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


@pytest.mark.parametrize("L", [3, 100])
def test_commit_slabs_that_layers_share(cuda_device, L):
    """Layers that read one another's slabs name them again: each is moved once, whichever layers and whichever of K and V name it."""
    rng = random.Random(L)
    T, N, Hkv = 24, 3, 2
    some = slabs(cuda_device, 5, N, Hkv, T + 40, 64, "f16", 7)
    before = [x.clone() for x in some]
    k = [some[(0, 0, 1, 2)[i % 4]] for i in range(L)]
    v = [some[(3, 3, 4, 2)[i % 4]] for i in range(L)]
    if L == 3:
        k[2], v[2] = some[4], some[0]
    used = {x.data_ptr() for x in k + v}
    path = torch.tensor([rising(rng, T, 11)] * N, dtype=torch.int32, device=cuda_device)
    n_path, lens = (torch.tensor(x, dtype=torch.int32, device=cuda_device) for x in ([11] * N, [0, 7, 33]))
    want, want_len = R.commit(before, path, n_path, lens)
    got = mm3fa.DraftTree(torch.full((N, T), -1, dtype=torch.int32, device=cuda_device)).commit(mm3fa.CacheLayers(k, v), path, n_path, lens)
    assert torch.equal(got, want_len)
    for x, old, w in zip(some, before, want):
        assert torch.equal(x, w if x.data_ptr() in used else old)


@pytest.mark.parametrize("draft", [None, "f32"])
@pytest.mark.parametrize("V", [300, 5003, 40000])
@pytest.mark.parametrize("temperature", [2e-5, 1e-7, 1e6, 1e36, 3e38])
def test_verify_temperatures(cuda_device, temperature, V, draft):
    """From ones at which all but the largest logits vanish to ones at which every logit above -inf weighs the same."""
    def edit(s, par):
        x = s["logits"]
        x[:, :, ::7] = float("-inf")
        x[1] *= 1e4
        x[2] -= 1e4
        s["tokens"][3:, 1:] = x[3:, 0].argmax(-1)[:, None].to(torch.int32)
        s["tokens"][5, 1:], s["accept"][5] = 14, 0.0  # a token of no probability, whatever the number
    check_verify(cuda_device, 9, 12, V, "f32", draft, temperature, seed=V, edit=edit)
