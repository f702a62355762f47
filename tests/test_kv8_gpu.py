"""The 8-bit paged cache's operators on the GPU against plain references in 64 bits (tests/kv8_ref.py).

Codes, scales, tables, counts and copies have to be equal bit for bit: their definitions leave no
choice.  Attention is held to a bound of its arithmetic, derived in kv8_ref.attend from the inputs.
"""
import numpy as np
import pytest
import torch

import kv8_ref as R
import mm3fa
from mm3fa import ggml

pytestmark = pytest.mark.gpu

I32 = torch.int32
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def ints(*v, dev="cuda"):
    return torch.tensor(v, dtype=I32, device=dev)


# ---------------------------------------------------------------- attention

def repeats(st, rows):
    """How often a batch is repeated so that the kernel for many rows takes its `rows` rows per kv head (0: never): five
    units of 16 rows for every two SMs and each wave of CTAs of 128 rows."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    heads, units, tiles = st.N * st.Hkv, -(-rows // 16), -(-rows // 128)
    return next((r for r in range(1, 400) if 2 * r * heads * units >= 5 * sms * -(-r * heads * tiles // sms)), 0) if st.D <= 128 else 0


def many(st, rows):
    """`st` with its sequences repeated where that brings the kernel for many rows."""
    r = max(1, repeats(st, rows))
    st.table, st.len, st.N = st.table.repeat(r, 1), st.len.repeat(r), st.N * r
    return st


def run_attend(st, H, n_q, dtype, out_dtype=None, q=None, q_len=None, causal=True, softcap=0.0, scale=None, layer=0,
               what=""):
    q = st.randn(st.N, n_q, H, st.D).to(dtype).transpose(1, 2) if q is None else q
    scale = st.D ** -0.5 if scale is None else scale
    out = torch.full((st.N, n_q, H, st.D), 7.0, dtype=out_dtype or dtype, device="cuda")
    ql = None if q_len is None else ints(*q_len)
    st_cache = st.cache()
    st_cache.attend(layer, q, st.table, st.len, scale, out=out, q_len=ql, causal=causal, logit_softcap=softcap)
    first = out.clone()
    st_cache.attend(layer, q, st.table, st.len, scale, out=out, q_len=ql, causal=causal, logit_softcap=softcap)
    st_cache.check()
    assert torch.equal(first, out), f"{what}: two runs differ"
    ref, f32, p16 = R.attend(st, layer, q, scale, ql, causal, softcap, out=torch.full_like(out, 7.0).float())
    R.check_attend(out, ref, f32, p16, out.dtype, what)
    reps = repeats(st, H // st.Hkv * n_q)
    if reps > 1:  # the other kernel
        both = torch.full_like(out, 7.0).repeat(reps, 1, 1, 1)
        st_cache.attend(layer, q.repeat(reps, 1, 1, 1), st.table.repeat(reps, 1), st.len.repeat(reps), scale, out=both,
                        q_len=None if ql is None else ql.repeat(reps), causal=causal, logit_softcap=softcap)
        st_cache.check()
        R.check_attend(both[:st.N], ref, f32, p16, out.dtype, what)
        assert torch.equal(both, both[:st.N].repeat(reps, 1, 1, 1)), f"{what}: copies of a batch differ"
    return out


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("D,P", [(64, 16), (64, 128), (128, 16), (128, 32), (128, 64), (128, 128), (256, 16), (256, 64)])
def test_attend_sizes(cuda_device, D, P, dtype):
    st = R.State([1, 2, P - 1, P, P + 1, 313, 0, 700], 2, D, P, seed=D + P, device=cuda_device)
    run_attend(st, 8, 1, DTYPES[dtype])


@pytest.mark.parametrize("G", [1, 2, 3, 5, 7, 8, 9, 16, 17, 20])
def test_attend_head_ratios(cuda_device, G):
    st = R.State([130, 77], 3, 128, 64, seed=G, device=cuda_device)
    run_attend(st, 3 * G, 1, torch.float32)
    run_attend(st, 3 * G, 1, torch.bfloat16)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("n_q", [2, 5, 16, 33, 64, 100, 257])
def test_attend_rows_causal(cuda_device, n_q, dtype):
    """Causal rows, some of them before the first key (no key: zeros)."""
    st = R.State([n_q, n_q + 200, 500, max(1, n_q - 3), 0], 2, 128, 32, seed=n_q, device=cuda_device)
    out = run_attend(st, 8, n_q, DTYPES[dtype])
    assert (out[3, :min(3, n_q - 1)] == 0).all() and (out[4] == 0).all()
    run_attend(st, 8, n_q, DTYPES[dtype], causal=False)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("n_q,q_len", [(7, [7, 0, 1, 3]), (150, [150, 0, 1, 70]), (150, [-4, 200, 149, 128])])
def test_attend_ragged_rows_leave_the_rest(cuda_device, n_q, q_len, D):
    """Rows behind q_len keep their values (7.0 in the reference too)."""
    st = R.State([400, 20, 1, 600], 2, D, 64, seed=n_q, device=cuda_device)
    for dt in (torch.float32, torch.bfloat16):
        out = run_attend(st, 4, n_q, dt, q_len=q_len)
        for s, m in enumerate(q_len):
            assert (out[s, max(m, 0):] == 7.0).all()


@pytest.mark.parametrize("n_q", [1, 130])
def test_attend_missing_pages(cuda_device, n_q):
    """Entries outside the pool name no page: their keys are absent, rows that see no other become zeros."""
    st = R.State([400, 400, 64], 2, 128, 32, seed=5, device=cuda_device)
    st.table[0, 3] = -1
    st.table[0, 7] = st.n_pages
    st.table[0, 9] = 2 ** 31 - 1
    st.table[1, 0] = -2 ** 31
    st.table[2, :] = -1
    out = run_attend(st, 4, n_q, torch.float32)
    assert (out[2] == 0).all()
    run_attend(st, 4, n_q, torch.float16)


@pytest.mark.parametrize("n_q", [1, 70])
def test_attend_length_beyond_the_table(cuda_device, n_q):
    """Lengths are clamped to the table's tokens, negative ones to none."""
    st = R.State([128, 64, 10], 2, 64, 64, seed=6, device=cuda_device)
    st.len = ints(2 ** 31 - 1, -5, 10)
    run_attend(st, 4, n_q, torch.float32, causal=False)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("n_q", [1, 90])
def test_attend_softcap(cuda_device, n_q, dtype):
    st = R.State([300, 90], 2, 128, 64, seed=8, device=cuda_device)
    q = (st.randn(2, 8, n_q, 128) * 6).to(DTYPES[dtype])
    run_attend(st, 8, n_q, DTYPES[dtype], q=q, softcap=5.0)
    run_attend(st, 8, n_q, DTYPES[dtype], q=q, softcap=1e-3)


@pytest.mark.parametrize("n_q", [1, 80])
def test_attend_result_type(cuda_device, n_q):
    """16-bit queries with an F32 result."""
    st = R.State([300, 90], 2, 128, 64, seed=9, device=cuda_device)
    for dt in (torch.float16, torch.bfloat16):
        run_attend(st, 8, n_q, dt, out_dtype=torch.float32)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("n_q", [1, 3, 66])
def test_attend_strides(cuda_device, n_q, dtype):
    """Queries at odd offsets and strides, results inside a larger buffer, a table that is a slice, layers."""
    st = many(R.State([200, 99], 2, 64, 32, L=3, seed=10, device=cuda_device), 2 * n_q)
    dt, n = DTYPES[dtype], st.N
    flat = st.randn(n * 4 * n_q * 77 + 1).to(dt)
    q = flat[1:].view(n, 4, n_q, 77)[..., 3:67]
    big = torch.full((n, n_q + 2, 9, 65), 7.0, dtype=dt, device=cuda_device)
    out = big[:, 1:n_q + 1, 2:6, 1:]
    wide = torch.full((n, st.table.shape[1] + 5), -7, dtype=I32, device=cuda_device)
    wide[:, 2:2 + st.table.shape[1]] = st.table
    table = wide[:, 2:2 + st.table.shape[1]]
    c = st.cache()
    c.attend(2, q, table, st.len, 0.125, out=out)
    ref, f32, p16 = R.attend(st, 2, q, 0.125)
    R.check_attend(out, ref, f32, p16, dt)
    rest = big.clone()
    rest[:, 1:n_q + 1, 2:6, 1:] = 7.0
    assert (rest == 7.0).all()


@pytest.mark.parametrize("n_q", [1, 65])
def test_attend_scales_of_every_size(cuda_device, n_q):
    """Value scales from 0 over 1e-38 to 1e30 in one sequence, and key scales that make a few keys win."""
    for seed, vs in ((1, [1e-3, 0.0, 2e-3, 1e-30, 1e-3]), (2, [1e-38, 0.0, 3e-38, 1e-38, 2e-38]),
                     (3, [1e30, 1e-30, 0.0, 1.0, 1e20]), (4, [0.0] * 5), (5, [1e-44, 1e-3, 1e-44, 1e-3, 0.0])):
        st = R.State([300, 37], 2, 128, 64, seed=seed, device=cuda_device)
        st.vs[0, st.table[0, :5].long()] = torch.tensor(vs, device=cuda_device)[:, None]
        st.ks[0, st.table[0, 2].long()] = 0.5
        run_attend(st, 8, n_q, torch.float32, what=f"scales {vs}")


@pytest.mark.parametrize("n_q", [1, 65])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attend_large_and_small_queries(cuda_device, n_q, dtype):
    """Queries far outside F16's range, with a scale that brings the scores back."""
    st = R.State([300, 37], 2, 128, 64, seed=12, device=cuda_device)
    q = st.randn(2, 8, n_q, 128)
    for f in (1e9, 1e-9, 1e30, 1e-30):
        run_attend(st, 8, n_q, DTYPES[dtype], q=(q * f).to(DTYPES[dtype]), scale=0.1 / f, what=f"queries times {f}")
    # a row whose elements span many powers of two, and rows of zeros
    wide = q * torch.exp2(torch.linspace(-30, 0, 128, device=cuda_device))
    wide[:, 1] = 0
    run_attend(st, 8, n_q, DTYPES[dtype], q=wide.to(DTYPES[dtype]), scale=0.3)


@pytest.mark.parametrize("n_q", [1, 65])
def test_attend_sharp_and_ordered_scores(cuda_device, n_q):
    """One key far above the rest, at the start or the end, and scores that rise with every key."""
    st = R.State([700, 700, 700], 1, 64, 64, seed=13, device=cuda_device)
    st.k.zero_()
    st.ks.fill_(1.0)
    st.vs.fill_(0.01)
    for s, f in enumerate((lambda t: 100 if t == 3 else 0, lambda t: 100 if t == 600 else -100, lambda t: t % 700 // 6 - 60)):
        for t in range(700):
            st.k[0, int(st.table[s, t // 64]), 0, t % 64, 0] = f(t)
    q = torch.zeros(3, 4, n_q, 64, device=cuda_device)
    q[..., 0] = 1.0
    run_attend(st, 4, n_q, torch.float32, q=q, scale=1.0)
    run_attend(st, 4, n_q, torch.float16, q=q.half(), scale=1.0)


@pytest.mark.parametrize("n_q", [1, 65])
def test_attend_nan_stays_in_its_rows(cuda_device, n_q):
    st = many(R.State([300, 37], 2, 64, 64, seed=14, device=cuda_device), 2 * n_q)
    q = st.randn(st.N, 4, n_q, 64)
    good = torch.empty(st.N, n_q, 4, 64, device=cuda_device)
    st.cache().attend(0, q, st.table, st.len, 0.125, out=good)
    for bad in (float("nan"), float("inf")):
        q2, out = q.clone(), torch.empty_like(good)
        q2[0, 1, n_q - 1, 5] = bad
        st.cache().attend(0, q2, st.table, st.len, 0.125, out=out)
        assert out[0, n_q - 1, 1].isnan().all()
        out[0, n_q - 1, 1] = good[0, n_q - 1, 1]
        assert torch.equal(out, good)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_attend_rows_that_grow_beside_rows_that_start_late(cuda_device, dtype):
    """Many rows whose scores rise by far from tile to tile beside causal rows that see no key yet, and beside rows
    of NaN: each takes its maxima up when it needs to, whatever its neighbours do."""
    dt = DTYPES[dtype]
    st = R.State([600, 520], 1, 64, 64, seed=17, device=cuda_device)
    st.k.zero_()
    st.ks.fill_(1.0)
    for s, n in enumerate((600, 520)):
        for j in range(-(-n // 64)):
            st.k[0, int(st.table[s, j]), 0, :, 0] = 12 * j  # 12 units of 2^s more each page
    q = torch.zeros(2, 4, 130, 64, device=cuda_device)
    q[..., 0] = torch.linspace(-2, 2, 130, device=cuda_device)
    q = q.to(dt)
    run_attend(st, 4, 130, dt, q=q, scale=1.0)
    run_attend(st, 4, 130, dt, q=q, scale=1.0, causal=False)
    many(st, 4 * 130)
    q = q.repeat(st.N // 2, 1, 1, 1)
    want = st.cache().attend(0, q, st.table, st.len, 1.0)
    q2 = q.clone()
    q2[0, :, 5::8] = float("nan")
    got = st.cache().attend(0, q2, st.table, st.len, 1.0)
    assert got[0, 5::8].isnan().all()
    got[0, 5::8] = want[0, 5::8]
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("n_q", [1, 130])
def test_attend_one_score_far_above_those_before(cuda_device, n_q, dtype):
    """In a later block of keys a single key far above all before it (2^s up to 2^30000), at every place of a page."""
    st = R.State([300], 1, 64, 16, seed=21, device=cuda_device)
    st.ks.fill_(1.0)
    st.k[..., 0] = 0
    q = torch.zeros(1, 2, n_q, 64, device=cuda_device)
    q[..., 1] = 0.01
    for at in (160, 161, 162, 175, 271):
        for jump in (1.0, 1.25, 2.0, 100.0):
            st.k[0, int(st.table[0, at // 16]), 0, at % 16, 0] = 127
            q[..., 0] = jump
            run_attend(st, 2, n_q, DTYPES[dtype], q=q.to(DTYPES[dtype]), scale=1.0, causal=False, what=f"{at} {jump}")
            st.k[..., 0] = 0


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("D", [64, 128])
def test_attend_many_rows_over_long_caches(cuda_device, D, dtype):
    """Some hundred rows over long caches, whose keys are split: sequences of many parts beside ones of one, of none, with
    missing pages, rows that see nothing of the last parts, ragged rows."""
    dt = DTYPES[dtype]
    st = R.State([5000, 130, 0, 2600], 2, D, 64, seed=22, device=cuda_device)
    run_attend(st, 8, 64, dt)
    run_attend(st, 8, 64, dt, causal=False, softcap=3.0)
    run_attend(st, 8, 90, dt, q_len=[90, 33, 5, 70])
    st.table[0, 20:50] = -1
    run_attend(st, 8, 64, dt)
    st = R.State([5000], 1, D, 32, seed=23, device=cuda_device)
    run_attend(st, 1, 1200, dt)
    run_attend(st, 3, 1000, dt, q_len=[999])
    st.vs[0, st.table[0, :120].long()] *= 1e-30  # the first parts' values are far below the last's
    st.ks[0, st.table[0, 130:].long()] *= 20
    run_attend(st, 3, 1000, dt, causal=False)


@pytest.mark.parametrize("D", [64, 128])
def test_attend_units_as_long_as_each_other(cuda_device, D):
    """About as many units as CTAs, of more than a few blocks: whole units for each."""
    for n in (50, 57, 110):
        st = R.State([600 + 5 * i for i in range(n)], 8, D, 64, seed=n, device=cuda_device)
        run_attend(st, 16, 1, torch.bfloat16)


@pytest.mark.parametrize("N,H,Hkv,n_q", [(300, 4, 2, 1), (65, 2, 1, 40), (1, 64, 32, 1)])
def test_attend_many_sequences(cuda_device, N, H, Hkv, n_q):
    st = R.State([(37 * i) % 211 for i in range(N)], Hkv, 64, 16, seed=N, device=cuda_device)
    run_attend(st, H, n_q, torch.float32)


def test_attend_long(cuda_device):
    """A long cache, split over many blocks, next to a short one; values of one sign (sums that only grow)."""
    st = R.State([20001, 3, 9999], 2, 128, 64, seed=15, device=cuda_device)
    st.v.abs_()
    run_attend(st, 8, 1, torch.float32)
    run_attend(st, 8, 1, torch.bfloat16)
    run_attend(st, 8, 70, torch.float32)
    run_attend(st, 8, 70, torch.float16)


@pytest.mark.parametrize("n_q", [1, 130])
def test_attend_streams_and_graph(cuda_device, n_q):
    """Two streams at once with a workspace each, then a graph that is replayed with other lengths and queries."""
    st = R.State([500, 1200], 4, 128, 64, seed=16, device=cuda_device)
    c = st.cache()
    q = st.randn(2, 16, n_q, 128)
    want = c.attend(0, q, st.table, st.len, 0.1).clone()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for i in range(20):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(c.attend(0, q, st.table, st.len, 0.1))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    graph, out = torch.cuda.CUDAGraph(), torch.empty_like(want)
    with torch.cuda.graph(graph):
        c.attend(0, q, st.table, st.len, 0.1, out=out)
    for lens in ((500, 1200), (1, 0), (333, 1199)):
        st.len.copy_(ints(*lens))
        q.copy_(st.randn(2, 16, n_q, 128))
        graph.replay()
        eager = c.attend(0, q, st.table, st.len, 0.1)
        torch.cuda.synchronize()
        assert torch.equal(eager, out)
        ref, f32, p16 = R.attend(st, 0, q, 0.1)
        R.check_attend(out, ref, f32, p16, torch.float32)


def test_one_workspace_for_every_shape(cuda_device):
    """Calls of different head dims and rows take turns with one workspace: the counters of one are not another's."""
    cs = [R.State([9000, 7000], 8, D, 64, seed=D, device=cuda_device) for D in (128, 64, 256)]
    shapes = [(st, n_q, dt) for st in cs for n_q in (1, 4, 2, 30) for dt in (torch.bfloat16, torch.float32)]
    qs = [st.randn(2, 32, n_q, st.D).to(dt) for st, n_q, dt in shapes]
    want = [st.cache().attend(0, q, st.table, st.len, 0.1) for (st, _, _), q in zip(shapes, qs)]
    ws = torch.zeros(max(st.cache().attend_workspace(q, st.table) for (st, _, _), q in zip(shapes, qs)), dtype=torch.uint8,
                     device=cuda_device)
    ws[1 << 16:] = 255  # only the first 64 KiB have to be zero
    order = torch.randperm(4 * len(shapes), generator=torch.Generator().manual_seed(1)).tolist()
    for i in order:
        i %= len(shapes)
        st = shapes[i][0]
        out = torch.full_like(want[i], 7.0)
        st.cache().attend(0, qs[i], st.table, st.len, 0.1, out=out, ws=ws)
        assert torch.equal(out, want[i]), shapes[i][1:]


@pytest.mark.parametrize("n_q", [1, 70])
@pytest.mark.parametrize("scale", [-0.3, 0.0])
def test_attend_negative_and_zero_scales(cuda_device, n_q, scale):
    """A softmax scale of 0 or below, and pages whose key or value scale is negative or 0."""
    st = R.State([300, 90], 2, 128, 64, seed=18, device=cuda_device)
    for dt in (torch.float32, torch.bfloat16):
        run_attend(st, 8, n_q, dt, scale=scale)
    st.ks[0, st.table[0, 1].long()] *= -1
    st.ks[0, st.table[0, 2].long()] = 0
    st.vs[0, st.table[0, 3].long()] *= -1
    for dt in (torch.float32, torch.float16, torch.bfloat16):
        run_attend(st, 8, n_q, dt, scale=scale)
        run_attend(st, 8, n_q, dt, scale=0.2)


def test_on_a_given_stream(cuda_device):
    """Calls on a stream that is not the current one: results and workspaces are made there."""
    st = R.State([500, 1200], 4, 128, 64, room=[510, 1210], seed=19, device=cuda_device)
    q, x = st.randn(2, 16, 1, 128), st.randn(2, 4, 1, 128)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    c = st.cache()
    c.append(0, x, x, st.table, st.len, stream=side)
    got = c.attend(0, q, st.table, st.len + 1, 0.1, stream=side)
    side.synchronize()
    c.check(side)
    assert torch.equal(got, c.attend(0, q, st.table, st.len + 1, 0.1))


def test_offsets_beyond_32_bits(cuda_device):
    """A pool of more than 2^31 codes (and scales far into it): the last pages give what a small pool gives."""
    D, P, Hkv, n_pages = 128, 128, 8, 2 ** 31 // (128 * 128 * 8) + 40
    small = R.State([300, 129], Hkv, D, P, room=[500, 300], seed=20, device=cuda_device)
    k, v = (torch.zeros(1, n_pages, Hkv, P, D, dtype=torch.int8, device=cuda_device) for _ in range(2))
    ks, vs = (torch.zeros(1, n_pages, Hkv, device=cuda_device) for _ in range(2))
    off = n_pages - small.n_pages
    for big, little in ((k, small.k), (v, small.v), (ks, small.ks), (vs, small.vs)):
        big[:, off:] = little
    table = torch.where(small.table >= 0, small.table + off, -1)
    c, s = mm3fa.Kv8Cache(k, v, ks, vs), small.cache()
    x = small.randn(2, Hkv, 100, D)
    for cache, t in ((c, table), (s, small.table)):
        cache.append(0, x, x, t, small.len)
    assert torch.equal(k[:, off:], small.k) and torch.equal(ks[:, off:], small.ks) and not k[:, :off].any()
    n = small.len + 100
    for n_q in (1, 100):
        for dt in (torch.float32, torch.bfloat16):
            q = small.randn(2, 32, n_q, D).to(dt)
            assert torch.equal(c.attend(0, q, table, n, 0.1), s.attend(0, q, small.table, n, 0.1))
    ko, vo, k1, v1 = (torch.zeros(2, Hkv, 400, D, device=cuda_device) for _ in range(4))
    c.read(0, ko, vo, table, torch.zeros_like(n), n)
    s.read(0, k1, v1, small.table, torch.zeros_like(n), n)
    assert torch.equal(ko, k1) and torch.equal(vo, v1)
    refs = torch.zeros(n_pages, dtype=I32, device=cuda_device)
    refs[table[table >= 0].long()] = 1
    refs[:off] = 1  # the only free pages are far into the pool
    t2, l2, r2 = torch.empty_like(table), torch.empty_like(n), torch.empty_like(refs)
    c.fork(ints(0), ints(1), table, n, refs, t2, l2, r2)
    c.check()
    last = int(t2[1, 3])
    assert last >= off and int(refs[last]) == 0 and t2[1, :3].tolist() == table[0, :3].tolist()
    assert torch.equal(k[0, last], k[0, int(table[0, 3])]) and torch.equal(vs[0, last], vs[0, int(table[0, 3])])


# ---------------------------------------------------------------- append and read

def append_ref(st, layer, k, v, start, n_new):
    out = []
    for codes, scales, x in ((st.k, st.ks, k), (st.v, st.vs, v)):
        c, s, x = codes[layer].cpu().numpy().copy(), scales[layer].cpu().numpy().copy(), x.float().cpu().numpy()
        for i in range(st.N):
            n = x.shape[2] if n_new is None else max(0, min(int(n_new[i]), x.shape[2]))
            R.append_one(c, s, x[i], st.table[i].tolist(), int(start[i]), n, st.P)
        out += [c, s]
    return out


def check_append(st, k, v, start, n_new=None, layer=0):
    want = append_ref(st, layer, k, v, start, n_new)
    others = [t.clone() for t in (st.k, st.v, st.ks, st.vs)]
    st.cache().append(layer, k, v, st.table, ints(*start), None if n_new is None else ints(*n_new))
    got = [t[layer].cpu().numpy() for t in (st.k, st.ks, st.v, st.vs)]
    for name, g, w in zip(("k", "k_scale", "v", "v_scale"), got, want):
        assert np.array_equal(g, w), f"{name}: {(g != w).sum()} of {g.size} differ"
    for now, before in zip((st.k, st.v, st.ks, st.vs), others):
        for l in range(st.L):
            assert l == layer or torch.equal(now[l], before[l])


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("D,P", [(64, 16), (128, 32), (128, 64), (256, 128), (64, 128)])
@pytest.mark.parametrize("T", [1, 2, 63, 300])
def test_append(cuda_device, D, P, T, dtype):
    start = [0, 1, P - 1, P, 5 * P + 3]
    st = R.State(start, 2, D, P, L=2, room=[s + T for s in start], seed=T + P, device=cuda_device)
    k = (st.randn(5, T, 2, D) * 2).to(DTYPES[dtype]).transpose(1, 2)
    v = (st.randn(5, T, 2, D) * torch.exp(st.randn(5, 1, 2, 1))).to(DTYPES[dtype]).transpose(1, 2)
    check_append(st, k, v, start, layer=1)


def test_append_token_by_token(cuda_device):
    """A page filled one row at a time, the rows growing, so that the codes held are rounded again and again."""
    st = R.State([0, 17], 2, 64, 32, room=[96, 96], seed=3, device=cuda_device)
    for t in range(40):
        x = st.randn(2, 2, 1, 64) * (1.05 ** t)
        check_append(st, x, x * 0.5, [t, 17 + t])


def test_append_ragged_and_refused_rows(cuda_device):
    """n_new per sequence, a negative start, missing pages and rows behind the table are skipped."""
    st = R.State([10, 20, 30, 40, 50, 60], 2, 64, 16, room=[100] * 6, seed=4, device=cuda_device)
    st.table[3, 4] = -1
    st.table[3, 5] = st.n_pages
    x = st.randn(6, 2, 40, 64)
    check_append(st, x, x, [10, 20, -1, 40, 50, 100], n_new=[40, 0, 40, 40, -3, 99])


def test_append_rounding_and_special_values(cuda_device):
    """Ties, NaN, infinities, zeros, denormals and the largest numbers."""
    D, P = 64, 16
    st = R.State([0] * 8, 1, D, P, room=[32] * 8, seed=5, device=cuda_device)
    x = torch.zeros(8, 1, 16, D, device=cuda_device)
    half = torch.arange(16 * D, device=cuda_device).remainder(254).float() - 126.5
    x[0, 0] = half.view(16, D)
    x[0, 0, 0, 0] = 127.0                     # scale 1: every value a tie
    x[1, 0] = half.view(16, D) * 1e-42        # denormals
    x[2, 0] = half.view(16, D) * 2.6e36       # near the largest
    x[3] = st.randn(1, 16, D)
    x[3, 0, 0, :4] = torch.tensor([float("nan"), float("inf"), -float("inf"), 3.0])
    x[4, 0, 0, :2] = torch.tensor([float("inf"), float("nan")])  # nothing finite but zeros
    x[5, 0] = half.view(16, D) * 1e-45
    x[6, 0] = st.randn(16, D) * torch.exp2(torch.linspace(-140, 100, D, device=cuda_device))
    x[7, 0, 0, 0] = -3e38
    check_append(st, x, -x, [0] * 8)
    # rows behind them, with the scales that they left
    check_append(st, x.flip(0), x, [7] * 8)


def test_append_many_quotients(cuda_device):
    """A million quotients next to ties: x = (k + 1/2) d and its neighbours for scales that are not powers of two."""
    st = R.State([0] * 64, 1, 256, 64, room=[64] * 64, seed=6, device=cuda_device)
    x = torch.empty(64, 1, 64, 256, device=cuda_device)
    top = torch.exp(st.randn(64, 1, 1, 1))
    d = top / torch.tensor(127.0, device=cuda_device)
    kk = torch.randint(-126, 126, x.shape, generator=st.g).to(cuda_device) + 0.5
    x = kk * d
    n = torch.randint(-2, 3, x.shape, generator=st.g, dtype=I32).to(cuda_device)
    x = (x.view(I32) + n).view(torch.float32)
    x[:, :, 0, 0] = top[:, 0, 0, 0][:, None]
    check_append(st, x, x.flip(2), [0] * 64)


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_append_and_read_strides(cuda_device, dtype):
    dt = DTYPES[dtype]
    st = R.State([5, 33], 3, 64, 32, room=[60, 60], seed=7, device=cuda_device)
    flat = st.randn(2 * 3 * 20 * 67 + 1).to(dt)
    x = flat[1:].view(2, 3, 20, 67)[..., 2:66]
    check_append(st, x, x[:, :, :1].expand(2, 3, 20, 64), [5, 33])
    big = torch.full((2, 25, 4, 65), 7.0, dtype=dt, device=cuda_device)
    out = big[:, 2:22, 1:, 1:].transpose(1, 2)
    vout = torch.full((2, 3, 20, 64), 7.0, dtype=dt, device=cuda_device)
    st.cache().read(0, out, vout, st.table, ints(5, 33), ints(20, 13))
    for s, (a, n) in enumerate(((5, 20), (33, 13))):
        for res, pool, sc in ((out, st.k, st.ks), (vout, st.v, st.vs)):
            want, _ = R.keys_of(pool[0], sc[0], st.table[s], 60, st.n_pages)
            assert torch.equal(res[s, :, :n], want[:, a:a + n].float().to(dt))
            assert (res[s, :, n:] == 7.0).all()
    big[:, 2:22, 1:, 1:] = 7.0
    assert (big == 7.0).all()


def test_read_edges(cuda_device):
    """Rows before the first token, behind the table and in missing pages are left; the rest is exact."""
    st = R.State([64, 64, 64], 2, 128, 16, seed=8, device=cuda_device)
    st.table[1, 1] = -1
    k, v = (torch.full((3, 2, 50, 128), 7.0, device=cuda_device) for _ in range(2))
    st.cache().read(0, k, v, st.table, ints(-10, 0, 40))
    want, _ = R.keys_of(st.k[0], st.ks[0], st.table[0], 64, st.n_pages)
    assert (k[0, :, :10] == 7.0).all() and torch.equal(k[0, :, 10:], want[:, :40].float())
    want, _ = R.keys_of(st.v[0], st.vs[0], st.table[1], 64, st.n_pages)
    assert (v[1, :, 16:32] == 7.0).all() and torch.equal(v[1, :, :16], want[:, :16].float())
    assert torch.equal(v[1, :, 32:], want[:, 32:50].float())
    want, _ = R.keys_of(st.v[0], st.vs[0], st.table[2], 64, st.n_pages)
    assert torch.equal(v[2, :, :24], want[:, 40:].float()) and (v[2, :, 24:] == 7.0).all()


# ---------------------------------------------------------------- pages

def outs(st):
    return (torch.full_like(st.table, 99), torch.full_like(st.len, 99), torch.full_like(st.refs, 99))


def check_moves(st, before, moves):
    for name, b in zip(("k", "v", "ks", "vs"), before):
        want = b.clone()
        for a, to in moves:
            want[:, to] = b[:, a]
        assert torch.equal(getattr(st, name), want), name


def check_fork(st, src, dst, deep=False, P=None):
    want = R.fork(st.table.tolist(), st.len.tolist(), st.refs.tolist(), src, dst, st.P, deep)
    before = [t.clone() for t in (st.k, st.v, st.ks, st.vs)]
    t2, l2, r2 = outs(st)
    c = st.cache()
    c.fork(None if src is None else ints(*src), ints(*dst), st.table, st.len, st.refs, t2, l2, r2, deep=deep)
    if want[4]:
        with pytest.raises(mm3fa.MM3FAError) as e:
            c.check()
        assert e.value.status == mm3fa.ERR_PAGES
    c.check()
    assert t2.tolist() == want[0] and l2.tolist() == want[1] and r2.tolist() == want[2]
    check_moves(st, before, want[3])
    st.table, st.len, st.refs = t2, l2, r2
    return want


@pytest.mark.parametrize("deep", [False, True])
@pytest.mark.parametrize("D,P,Hkv,L", [(64, 16, 1, 1), (128, 64, 3, 5), (256, 32, 2, 36)])
def test_fork(cuda_device, D, P, Hkv, L, deep):
    st = R.State([3 * P + 5, 2 * P, 0, 1, 7 * P - 1, 2], Hkv, D, P, L=L, spare=40, seed=P, device=cuda_device)
    check_fork(st, [0, 0, 4], [2, 3, 5], deep)         # onto an empty one and used ones
    check_fork(st, [4, 0, 1], [0, 4, 1], deep)         # a swap, and onto itself
    check_fork(st, [1, 2, 9, -5, 3], [5, 5, 0, 1, 7], deep)  # dst twice, indices out of range
    check_fork(st, [-1, 5], [4, 2], deep)              # emptied
    check_fork(st, None, [0, 1, 2, 3, 4, 5], deep)     # all freed
    assert st.refs.abs().sum() == 0 and (st.table == -1).all()


def test_fork_shares_counts(cuda_device):
    """Many forks of one prompt and their release leave the counts as they were."""
    st = R.State([100] + [0] * 70, 2, 64, 16, spare=80, seed=1, device=cuda_device)
    start = st.refs.clone()
    check_fork(st, [0] * 70, list(range(1, 71)))
    assert int(st.refs.max()) == 71
    check_fork(st, None, list(range(1, 71)))
    assert torch.equal(st.refs, start)


def test_fork_without_enough_pages(cuda_device):
    st = R.State([33, 0, 0], 2, 64, 16, spare=2, seed=2, device=cuda_device)
    assert check_fork(st, [0, 0], [1, 2], deep=True)[4]
    assert not check_fork(st, [0, 0], [1, 2])[4]
    assert check_fork(st, [0], [1])[4]  # the pages that dst gives up are not given out in the same call


def test_status_left_in_an_outgrown_workspace(cuda_device):
    """A call that found too few pages is reported though a larger one came between it and the check."""
    c = mm3fa.Kv8Cache.allocate(1, 5300, 1, 16, 64, cuda_device)
    refs = torch.ones(5300, dtype=I32, device=cuda_device)
    for n in (2, 500):
        table = torch.full((n, 1), -1, dtype=I32, device=cuda_device)
        c.reserve(table, refs, torch.ones(n, dtype=I32, device=cuda_device))
        refs.zero_()
    with pytest.raises(mm3fa.MM3FAError) as e:
        c.check()
    assert e.value.status == mm3fa.ERR_PAGES
    c.check()


def test_status_of_captured_calls(cuda_device):
    """check reports what a replayed call found where the stream had a workspace before the capture, and reads no
    workspace that only a graph has written."""
    c = mm3fa.Kv8Cache.allocate(1, 4, 1, 16, 64, cuda_device)
    refs, table, one = torch.ones(4, dtype=I32, device=cuda_device), torch.full((1, 1), -1, dtype=I32, device=cuda_device), ints(1)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for g in graphs:
        with torch.cuda.graph(g, stream=side):
            c.reserve(table, refs, one)
        c.check(side)
        with torch.cuda.stream(side):
            g.replay()
            if g is graphs[0]:
                c.check()
                c.reserve(table, torch.zeros_like(refs), ints(0))  # makes the stream's workspace
            else:
                with pytest.raises(mm3fa.MM3FAError):
                    c.check()
    assert int(table[0, 0]) == -1


def test_fork_missing_pages_and_no_pairs(cuda_device):
    st = R.State([100, 50], 2, 64, 16, spare=9, seed=3, device=cuda_device)
    st.table[0, 2] = -1
    st.table[0, 5] = st.n_pages + 3
    check_fork(st, [0], [1], deep=True)
    check_fork(st, [], [])
    check_fork(st, [0], [1])


@pytest.mark.parametrize("n_pages", [1, 7, 1023, 8200, 20011])
def test_compact(cuda_device, n_pages):
    g = torch.Generator().manual_seed(n_pages)
    for share in (0.0, 0.3, 0.9, 1.0):
        st = R.State([], 1, 64, 16, L=2, spare=n_pages, seed=n_pages, device=cuda_device)
        st.N = 3
        st.refs = ((torch.rand(n_pages, generator=g) < share).to(I32) * torch.randint(1, 4, (n_pages,), generator=g, dtype=I32)).to(cuda_device)
        st.table = torch.randint(-2, n_pages + 2, (3, 50), generator=g, dtype=I32).to(cuda_device)
        want = R.compact(st.table.tolist(), st.refs.tolist())
        before = [t.clone() for t in (st.k, st.v, st.ks, st.vs)]
        t2, _, r2 = torch.full_like(st.table, 99), None, torch.full_like(st.refs, 99)
        c = st.cache()
        c.compact(st.table, st.refs, t2, r2)
        c.check()
        assert t2.tolist() == want[0] and r2.tolist() == want[1]
        check_moves(st, before, want[2])


def test_reserve(cuda_device):
    st = R.State([40, 0, 17, 100], 2, 64, 16, spare=30, seed=4, device=cuda_device)
    c = st.cache()
    for n_tok in ([41, 20, 17, 100], [56, 0, 100, 112], [0, -4, 33, 64]):
        want = R.reserve(st.table.tolist(), st.refs.tolist(), n_tok, st.P)
        c.reserve(st.table, st.refs, ints(*n_tok))
        c.check()
        assert st.table.tolist() == want[0] and st.refs.tolist() == want[1] and not want[2]
    for n_tok in ([113, 0, 0, 0], [112, 112, 112, 112]):  # a row too short, the pool too small
        table, refs = st.table.tolist(), st.refs.tolist()
        if n_tok[0] == 112:
            st.refs[st.refs == 0] = 1
            refs = st.refs.tolist()
        c.reserve(st.table, st.refs, ints(*n_tok))
        with pytest.raises(mm3fa.MM3FAError) as e:
            c.check()
        assert e.value.status == mm3fa.ERR_PAGES
        assert st.table.tolist() == table and st.refs.tolist() == refs


# ---------------------------------------------------------------- together

@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_song_from_prompt_to_candidates(cuda_device, dtype):
    """reserve, append and attend a prompt and tokens after it; fork candidates, append to each, free some,
    compact, and attend again: every result against the values that `read` gives back."""
    dt = DTYPES[dtype]
    L, Hkv, H, D, P, N = 2, 2, 8, 128, 32, 4
    c = mm3fa.Kv8Cache.allocate(L, 60, Hkv, P, D, cuda_device)
    g = torch.Generator().manual_seed(0)
    rand = lambda *s: torch.randn(*s, generator=g).to(cuda_device).to(dt)
    table = torch.full((N, 12), -1, dtype=I32, device=cuda_device)
    refs = torch.zeros(60, dtype=I32, device=cuda_device)
    length = torch.zeros(N, dtype=I32, device=cuda_device)

    def step(T, n_new):
        nonlocal length
        new = ints(*n_new)
        c.reserve(table, refs, length + new)
        for layer in range(L):
            k, v, q = rand(N, Hkv, T, D), rand(N, Hkv, T, D), rand(N, H, T, D)
            c.append(layer, k, v, table, length, new)
            out = torch.full((N, T, H, D), 7.0, dtype=dt, device=cuda_device)
            c.attend(layer, q, table, length + new, D ** -0.5, out=out, q_len=new)
            check(layer, q, out, length + new, new)
            # what the cache holds of the new rows: within half a code of them
            ko, vo = torch.zeros_like(k).float(), torch.zeros_like(v).float()
            c.read(layer, ko, vo, table, length, new)
            for s, n in enumerate(n_new):
                for x, got, sc in ((k, ko, c.k_scale), (v, vo, c.v_scale)):
                    top = sc[layer, table[s][table[s] >= 0].long()].max().item() if n else 0
                    assert (got[s, :, :n] - x[s, :, :n].float()).abs().max().item() <= 0.5001 * top if n else True
        length = length + new
        c.check()

    def check(layer, q, out, lens, q_len):
        st = type("S", (), {})()
        st.k, st.v, st.ks, st.vs, st.table, st.n_pages, st.P, st.Hkv = c.k, c.v, c.k_scale, c.v_scale, table, 60, P, Hkv
        ref, f32, p16 = R.attend(st, layer, q, D ** -0.5, q_len, True, 0.0, out=torch.full_like(out, 7.0).float(), kv_len=lens)
        R.check_attend(out, ref, f32, p16, dt)

    step(100, [100, 71, 0, 0])
    for _ in range(3):
        step(1, [1, 1, 0, 0])
    t2, l2, r2 = torch.empty_like(table), torch.empty_like(length), torch.empty_like(refs)
    c.fork(ints(0, 1), ints(2, 3), table, length, refs, t2, l2, r2)
    table, length, refs = t2, l2, r2
    step(2, [2, 1, 2, 1])
    step(1, [1, 1, 1, 1])
    t2, l2, r2 = torch.empty_like(table), torch.empty_like(length), torch.empty_like(refs)
    c.free(ints(0), table, length, refs, t2, l2, r2)
    t3, r3 = torch.empty_like(table), torch.empty_like(refs)
    c.compact(t2, r2, t3, r3)
    c.check()
    live = int((r3 > 0).sum())
    assert (r3[:live] > 0).all() and (r3[live:] == 0).all()
    table, length, refs = t3, l2, r3
    step(1, [0, 1, 1, 1])


def test_with_the_decode_prologue_and_the_f16_attention(cuda_device):
    """A decode step: the fused prologue's normed and rotated k (through an F16 row) into the 8-bit cache, attention
    over it, and the F16 attention over the values read back: both within their bounds of each other."""
    N, H, Hkv, D, P = 2, 32, 8, 128, 64
    st = R.State([200, 77], Hkv, D, P, room=[201, 78], seed=20, device=cuda_device)
    F32, F16 = ggml.GGML_TYPE_F32, ggml.GGML_TYPE_F16
    q_in, k_in, v_in = st.randn(N, H, D), st.randn(N, Hkv, D), st.randn(N, Hkv, D)
    ones, pos, rows = torch.ones(D, device=cuda_device), ints(200, 77), torch.zeros(N, dtype=torch.int64, device=cuda_device)
    k16, v16 = (torch.zeros(N, Hkv, 1, D, dtype=torch.float16, device=cuda_device) for _ in range(2))
    q = torch.empty(N, H, D, device=cuda_device)
    mk = lambda ty, ne, t: ggml.make(ty, ne, t.data_ptr())
    mm3fa.decode_prologue(mk(F32, [D, H, N], q_in), mk(F32, [D, Hkv, N], k_in), mk(F32, [D, Hkv, N], v_in), ones.data_ptr(),
                          ones.data_ptr(), 1e-6, pos.data_ptr(), 1e6, rows.data_ptr(), mk(F16, [D, 1, Hkv, N], k16),
                          mk(F16, [D, 1, Hkv, N], v16), mk(F32, [D, H, N], q), torch.cuda.current_stream().cuda_stream)
    c = st.cache()
    c.append(0, k16, v16, st.table, st.len)
    st.len = st.len + 1
    out = c.attend(0, q.view(N, H, 1, D), st.table, st.len, D ** -0.5)
    ref, f32, p16 = R.attend(st, 0, q.view(N, H, 1, D), D ** -0.5)
    R.check_attend(out, ref, f32, p16, torch.float32)
    n_kv = 256
    kf, vf = (torch.zeros(N, Hkv, n_kv, D, dtype=torch.float16, device=cuda_device) for _ in range(2))
    c.read(0, kf, vf, st.table, ints(0, 0), st.len)
    mask = torch.full((N, 1, 1, n_kv), float("-inf"), dtype=torch.float16, device=cuda_device)
    for s in range(N):
        mask[s, ..., :int(st.len[s])] = 0
    dst = torch.empty(N, 1, H, D, device=cuda_device)
    qd = ggml.make(F32, [D, 1, H, N], q.data_ptr())
    mm3fa.run(qd, ggml.from_torch(kf), ggml.from_torch(vf), ggml.from_torch(mask),
              ggml.make(F32, [D, H, 1, N], dst.data_ptr()), D ** -0.5)
    # the F16 path rounds q, k, v and the weights to 11 bits: 2^-11 each of values up to |v|, and of scores up to |s|
    vmax = vf.float().abs().max().item()
    big = (q.abs().sum(-1).max() * kf.float().abs().max() * D ** -0.5).item()
    assert (dst - out).abs().max().item() <= vmax * (2 * big * 2.0 ** -10 + 3 * 2.0 ** -11)
