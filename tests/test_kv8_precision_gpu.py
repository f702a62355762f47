"""How exact the attention over the 8-bit cache is, on the GPU, in bounds that do not grow with the number of keys
(tests/kv8_precision.py)."""
import pytest
import torch

import kv8_precision as E
import kv8_ref as R
from test_kv8_gpu import DTYPES, many, run_attend

pytestmark = pytest.mark.gpu


def attend(st, q, out_dtype=None, causal=True):
    out = None if out_dtype is None else torch.empty(q.shape[0], q.shape[2], q.shape[1], q.shape[3], dtype=out_dtype, device=q.device)
    c = st.cache()
    out = c.attend(0, q, st.table, st.len, st.D ** -0.5, out=out, causal=causal)
    c.check()
    return out


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("n_q", [1, 4, 16, 70])
def test_f32_results_keep_22_bits(cuda_device, n_q, D, dtype):
    """F32 results of queries of each type, from 64 keys to thousands."""
    st = R.State([64, 500, 3001], 2, D, 64, seed=25, device=cuda_device)
    q = st.randn(3, 8, n_q, D).to(DTYPES[dtype])
    copies = many(st, 4 * n_q).N // 3
    got = attend(st, q.repeat(copies, 1, 1, 1), torch.float32)
    st.table, st.len, st.N = st.table[:3], st.len[:3], 3
    E.check(st, q, got[:3], f"D {D}, {n_q} rows")


@pytest.mark.parametrize("n_q", [1, 70])
def test_f32_results_over_long_caches(cuda_device, n_q):
    """20001 keys, values of both signs and of one."""
    st = R.State([20001, 700, 9999], 2, 128, 64, seed=15, device=cuda_device)
    q = st.randn(3, 8, n_q, 128)
    E.check(st, q, attend(st, q), "both signs")
    st.v.abs_()
    E.check(st, q, attend(st, q), "one sign")


def one_large(st, n_q, x, dtype):
    """Queries with one element of +-x in a dimension where every key is 0, the others around 1."""
    q = st.randn(st.N, 8, n_q, st.D).to(dtype)
    q[..., 7] = torch.where(q[..., 7] > 0, x, -x)
    st.k[..., 7] = 0
    return q


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("n_q", [1, 4, 70])
@pytest.mark.parametrize("dtype,x", [("f16", 256), ("f16", 1000), ("f16", 60000), ("bf16", 1000), ("bf16", 1e5), ("bf16", 1e6), ("f32", 1000),
                                     ("f32", 1e5)])
def test_one_large_element_of_q(cuda_device, dtype, x, n_q, D):
    """The small elements beside a large one decide: its own products are 0."""
    dt = DTYPES[dtype]
    st = many(R.State([300, 90], 2, D, 64, seed=26, device=cuda_device), 4 * n_q)
    q = one_large(st, n_q, x, dt)
    got = attend(st, q)
    ref, f32, p16 = R.attend(st, 0, q, D ** -0.5)
    R.check_attend(got, ref, f32, p16, dt, f"one element of {x}")
    if dtype == "f32":
        E.check(st, q, got, f"one element of {x}")


@pytest.mark.parametrize("n_q", [1, 65])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("f", [1e-38, 1e-34, 1e-28, 1e36])
def test_queries_near_the_smallest_and_largest_numbers(cuda_device, f, dtype, n_q):
    """Rows that a power of two alone cannot bring to their place, with a scale that brings the scores back."""
    st = R.State([300, 37], 2, 128, 64, seed=12, device=cuda_device)
    run_attend(st, 8, n_q, DTYPES[dtype], q=(st.randn(2, 8, n_q, 128) * f).to(DTYPES[dtype]), scale=0.1 / f)


@pytest.mark.parametrize("N,n,H,D,n_q", [(64, 8000, 32, 128, 1), (64, 8000, 16, 64, 1), (20, 8000, 32, 128, 4), (32, 4000, 8, 256, 1),
                                         (16, 4000, 8, 256, 12)])
def test_f32_sums_over_many_long_sequences(cuda_device, N, n, H, D, n_q):
    """So many units that each CTA walks thousands of keys of one, with values of one sign: nothing is lost on the way."""
    st = R.State([n] * N, 8, D, 64, seed=34, device=cuda_device)
    st.v.abs_()
    q = st.randn(N, H, n_q, D)
    got = attend(st, q)
    st.table, st.len, st.N = st.table[:3], st.len[:3], 3
    E.check(st, q[:3], got[:3], f"{N} of {n}")


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("n_q", [1, 4, 70])
def test_tables_of_more_than_65536_tokens(cuda_device, n_q, D, dtype):
    """The sums that long tables get, in 16-bit results too."""
    st = R.State([300, 1000, 5], 2, D, 128, seed=35, device=cuda_device)
    wide = torch.full((3, 600), -1, dtype=torch.int32, device=cuda_device)
    wide[:, :st.table.shape[1]] = st.table
    st.table = wide
    run_attend(st, 8, n_q, DTYPES[dtype])
    run_attend(st, 8, n_q, DTYPES[dtype], softcap=4.0)
