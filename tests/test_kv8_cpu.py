"""What the 8-bit paged cache refuses, on host tensors: every check of the C ABI and of the Python class runs
before anything is launched (without a device an accepted call ends with ERR_DEVICE)."""
import types

import pytest
import torch

import kv8_ref
import mm3fa
from mm3fa import kv8

no_gpu = pytest.mark.skipif(torch.cuda.is_available(), reason="host tensors are accepted up to the device check only")


def status(fn, *a, **kw):
    with pytest.raises(mm3fa.MM3FAError) as e:
        fn(*a, **kw)
    return e.value.status


def make(**kw):
    kw = {"lens": [70, 5], "Hkv": 2, "D": 64, "P": 32, "room": [80, 40], **kw}
    return kv8_ref.State(**kw)


def test_cache_refusals():
    s = make()
    C = mm3fa.Kv8Cache
    assert status(C, s.k[0], s.v[0], s.ks[0], s.vs[0]) == mm3fa.ERR_SHAPE
    assert status(C, s.k, s.v, s.ks[:, :-1], s.vs) == mm3fa.ERR_SHAPE
    assert status(C, s.k.float(), s.v, s.ks, s.vs) == mm3fa.ERR_TYPE
    assert status(C, s.k, s.v, s.ks.double(), s.vs) == mm3fa.ERR_TYPE
    assert status(C, s.k.transpose(2, 3).contiguous().transpose(2, 3), s.v, s.ks, s.vs) == mm3fa.ERR_STRIDE


@no_gpu
@pytest.mark.parametrize("D,P", [(32, 32), (96, 32), (64, 8), (64, 48), (64, 256)])
def test_unsupported_sizes(D, P):
    c = mm3fa.Kv8Cache(torch.zeros(1, 4, 2, P, D, dtype=torch.int8), torch.zeros(1, 4, 2, P, D, dtype=torch.int8),
                       torch.zeros(1, 4, 2), torch.zeros(1, 4, 2))
    t, n = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    x = torch.zeros(1, 2, 1, D)
    assert status(c.append, 0, x, x, t, n) == mm3fa.ERR_UNSUPPORTED
    assert status(c.reserve, t, torch.zeros(4, dtype=torch.int32), n) == mm3fa.ERR_UNSUPPORTED
    assert c._call("pages_workspace", c._desc, 1) == 0


@no_gpu
def test_append_and_read_refusals():
    s = make()
    c, x = s.cache(), torch.zeros(2, 2, 3, 64)
    ok = status(c.append, 0, x, x, s.table, s.len)
    assert ok == mm3fa.ERR_DEVICE  # accepted but for the device
    assert status(c.read, 0, x, x, s.table, s.len) == mm3fa.ERR_DEVICE
    for layer in (-1, 1):
        assert status(c.append, layer, x, x, s.table, s.len) == mm3fa.ERR_SHAPE
    assert status(c.append, 0, x, x[:, :, :2], s.table, s.len) == mm3fa.ERR_SHAPE
    assert status(c.append, 0, x[:, :1], x[:, :1], s.table, s.len) == mm3fa.ERR_SHAPE
    assert status(c.append, 0, x[:1], x[:1], s.table, s.len) == mm3fa.ERR_SHAPE
    assert status(c.append, 0, x[:, :, :0], x[:, :, :0], s.table, s.len) == mm3fa.ERR_SHAPE
    assert status(c.append, 0, x[..., :32], x[..., :32], s.table, s.len) == mm3fa.ERR_SHAPE
    assert status(c.append, 0, x.double(), x, s.table, s.len) == mm3fa.ERR_TYPE
    assert status(c.append, 0, x, x, s.table, s.len.long()) == mm3fa.ERR_TYPE
    assert status(c.append, 0, x, x, s.table, s.len[:1]) == mm3fa.ERR_SHAPE
    assert status(c.append, 0, x, x, s.table.long(), s.len) == mm3fa.ERR_TYPE
    assert status(c.append, 0, x, x, s.table[0], s.len) == mm3fa.ERR_SHAPE
    assert status(c.append, 0, x, x, s.table.t().contiguous().t(), s.len) == mm3fa.ERR_STRIDE
    wide = torch.zeros(2, 2, 3, 128)[..., ::2]
    assert status(c.append, 0, wide, wide, s.table, s.len) == mm3fa.ERR_STRIDE
    # rows that are read may be broadcast, rows that are written may not
    one = torch.zeros(2, 2, 1, 64).expand(2, 2, 3, 64)
    assert status(c.append, 0, one, one, s.table, s.len) == mm3fa.ERR_DEVICE
    assert status(c.read, 0, one, x, s.table, s.len) == mm3fa.ERR_STRIDE


@no_gpu
def test_attend_refusals():
    s = make()
    c, q = s.cache(), torch.zeros(2, 4, 3, 64)
    out = torch.zeros(2, 3, 4, 64)
    ws = torch.zeros(1 << 20, dtype=torch.uint8)
    a = lambda *x, **kw: status(c.attend, *x, **{"ws": ws, **kw})
    assert a(0, q, s.table, s.len, 0.1, out) == mm3fa.ERR_DEVICE
    assert a(0, q.half(), s.table, s.len, 0.1, out) == mm3fa.ERR_DEVICE
    assert a(0, q.half(), s.table, s.len, 0.1, out.bfloat16()) == mm3fa.ERR_TYPE
    assert a(0, q, s.table, s.len, 0.1, out.half()) == mm3fa.ERR_TYPE
    assert a(0, q, s.table, s.len, 0.1, torch.zeros(2, 4, 3, 64)) == mm3fa.ERR_SHAPE
    assert a(0, torch.zeros(2, 3, 3, 64), s.table, s.len, 0.1, torch.zeros(2, 3, 3, 64)) == mm3fa.ERR_SHAPE
    assert a(0, q[:1], s.table, s.len, 0.1, out[:1]) == mm3fa.ERR_SHAPE
    assert a(1, q, s.table, s.len, 0.1, out) == mm3fa.ERR_SHAPE
    assert a(0, q, s.table, s.len, float("nan"), out) == mm3fa.ERR_SHAPE
    assert a(0, q, s.table, s.len, 0.1, out, logit_softcap=-1.0) == mm3fa.ERR_SHAPE
    assert a(0, q, s.table, s.len, 0.1, out, logit_softcap=float("inf")) == mm3fa.ERR_SHAPE
    assert a(0, q, s.table, s.len, 0.1, out, ws=ws[:16]) == mm3fa.ERR_WORKSPACE
    assert a(0, q, s.table, s.len, 0.1, out, ws=ws[8:]) == mm3fa.ERR_WORKSPACE
    assert a(0, q, s.table, s.len, 0.1, torch.zeros(2, 1, 4, 64).expand(2, 3, 4, 64)) == mm3fa.ERR_STRIDE
    assert status(c.attend, 0, q, s.table, s.len[:1], 0.1, out, ws=ws) == mm3fa.ERR_SHAPE
    assert status(c.attend, 0, q, s.table, s.len, 0.1, out, q_len=s.len[:1], ws=ws) == mm3fa.ERR_SHAPE
    # the C entry with pointers missing
    f, st = kv8._calls()["attn"], (1 << 20)
    qd, od, td = c._rows(q), c._rows(out), c._table(s.table)
    assert f(None, 0, qd, td, s.len.data_ptr(), None, 0.1, 0.0, 1, od, ws.data_ptr(), st, None) == mm3fa.ERR_NULL
    assert f(c._desc, 0, None, td, s.len.data_ptr(), None, 0.1, 0.0, 1, od, ws.data_ptr(), st, None) == mm3fa.ERR_NULL
    assert f(c._desc, 0, qd, td, None, None, 0.1, 0.0, 1, od, ws.data_ptr(), st, None) == mm3fa.ERR_NULL
    assert f(c._desc, 0, qd, td, s.len.data_ptr(), None, 0.1, 0.0, 1, od, None, st, None) == mm3fa.ERR_WORKSPACE


@no_gpu
def test_page_operation_refusals():
    s = make()
    c = s.cache()
    t2, l2, r2 = torch.empty_like(s.table), torch.empty_like(s.len), torch.empty_like(s.refs)
    pair = torch.tensor([0], dtype=torch.int32), torch.tensor([1], dtype=torch.int32)
    f = lambda *x, **kw: status(c.fork, *pair, *x, **kw)
    assert f(s.table, s.len, s.refs, t2, l2, r2) == mm3fa.ERR_DEVICE
    assert status(c.free, pair[1], s.table, s.len, s.refs, t2, l2, r2) == mm3fa.ERR_DEVICE
    # results in the inputs' own buffers
    assert f(s.table, s.len, s.refs, s.table, l2, r2) == mm3fa.ERR_UNSUPPORTED
    assert f(s.table, s.len, s.refs, t2, s.len, r2) == mm3fa.ERR_UNSUPPORTED
    assert f(s.table, s.len, s.refs, t2, l2, s.refs) == mm3fa.ERR_UNSUPPORTED
    both = torch.zeros(3, s.table.shape[1], dtype=torch.int32)
    assert f(both[:2], s.len, s.refs, both[1:], l2, r2) == mm3fa.ERR_UNSUPPORTED
    assert f(s.table, s.len, s.refs, t2[:1], l2, r2) == mm3fa.ERR_SHAPE
    assert f(s.table, s.len, s.refs[:-1], t2, l2, r2) == mm3fa.ERR_SHAPE
    assert f(s.table, s.len, s.refs.long(), t2, l2, r2) == mm3fa.ERR_TYPE
    assert status(c.fork, pair[0], pair[1].long(), s.table, s.len, s.refs, t2, l2, r2) == mm3fa.ERR_TYPE
    assert status(c.compact, s.table, s.refs, t2, r2) == mm3fa.ERR_DEVICE
    assert status(c.compact, s.table, s.refs, s.table, r2) == mm3fa.ERR_UNSUPPORTED
    assert status(c.compact, s.table, s.refs, t2, s.refs) == mm3fa.ERR_UNSUPPORTED
    assert status(c.reserve, s.table, s.refs, s.len) == mm3fa.ERR_DEVICE
    assert status(c.reserve, s.table, s.refs, s.len[:1]) == mm3fa.ERR_SHAPE
    # a workspace that is too small, an unknown flag
    g, ws = kv8._calls()["fork"], torch.zeros(1 << 20, dtype=torch.uint8)
    args = lambda flags, nbytes: g(c._desc, c._table(s.table), s.len.data_ptr(), s.refs.data_ptr(), pair[0].data_ptr(),
                                   pair[1].data_ptr(), 1, flags, c._table(t2), l2.data_ptr(), r2.data_ptr(),
                                   ws.data_ptr(), nbytes, None)
    need = c._call("pages_workspace", c._desc, 2)
    assert args(0, need) == mm3fa.ERR_DEVICE
    assert args(0, need - 1) == mm3fa.ERR_WORKSPACE
    assert args(2, need) == mm3fa.ERR_UNSUPPORTED

    # tables whose entries are not counted in 32 bits
    big = lambda pages: kv8._PACK_TABLE(s.table.data_ptr(), pages, pages, 65535)
    other = lambda pages: kv8._PACK_TABLE(t2.data_ptr() + (1 << 40), pages, pages, 65535)
    need = c._call("pages_workspace", c._desc, 65535)
    for pages, want in ((32768, mm3fa.ERR_DEVICE), (32769, mm3fa.ERR_UNSUPPORTED)):
        got = c._call("reserve", c._desc, big(pages), s.refs.data_ptr(), s.len.data_ptr(), ws.data_ptr(), need, None)
        assert got == want
        got = c._call("compact", c._desc, big(pages), s.refs.data_ptr(), other(pages), r2.data_ptr(), ws.data_ptr(), need, None)
        assert got == want


@no_gpu
def test_a_stream_of_another_device():
    s = make()
    c, x = s.cache(), torch.zeros(2, 2, 3, 64)
    other = types.SimpleNamespace(device_index=0, cuda_stream=0)
    with pytest.raises(ValueError):
        c.append(0, x, x, s.table, s.len, stream=other)
    with pytest.raises(ValueError):
        c.attend(0, x, s.table, s.len, 1.0, stream=other)
    with pytest.raises(ValueError):
        c.check(other)


def test_status_strings():
    assert "pages" in mm3fa.status_string(mm3fa.ERR_PAGES)
