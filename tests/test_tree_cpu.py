"""What the operators of tree decoding refuse, on host tensors: every check of the C ABI and of the Python classes runs
before anything is launched (without a device an accepted call ends with ERR_DEVICE)."""
import pytest
import torch

import mm3fa
from mm3fa import tree as T_

no_gpu = pytest.mark.skipif(torch.cuda.is_available(), reason="host tensors are accepted up to the device check only")
WS = torch.zeros(1 << 28, dtype=torch.uint8)


def status(fn, *a, **kw):
    with pytest.raises(mm3fa.MM3FAError) as e:
        fn(*a, **kw)
    return e.value.status


def ints(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def test_tree_refusals():
    assert status(mm3fa.DraftTree, ints(5)) == mm3fa.ERR_SHAPE
    assert status(mm3fa.DraftTree, ints(0, 5)) == mm3fa.ERR_SHAPE
    assert status(mm3fa.DraftTree, ints(2, 5).long()) == mm3fa.ERR_TYPE
    assert status(mm3fa.DraftTree, ints(5, 2).t()) == mm3fa.ERR_STRIDE
    assert status(mm3fa.DraftTree, ints(2, 5), ints(3)) == mm3fa.ERR_SHAPE
    assert status(mm3fa.DraftTree, ints(2, 5), ints(2).float()) == mm3fa.ERR_TYPE


@no_gpu
def test_attend_refusals():
    t = mm3fa.DraftTree(ints(1, 5))
    q, k, n = torch.zeros(2, 4, 5, 64), torch.zeros(2, 2, 30, 64, dtype=torch.float16), ints(2)
    a = lambda q=q, k=k, v=None, n=n, t=t, ws=WS, scale=0.1, **kw: status(t.attend, q, k, k if v is None else v, n, scale, ws=ws, **kw)
    assert a() == mm3fa.ERR_DEVICE  # accepted but for the device
    for ty in (torch.bfloat16, torch.float32):
        assert a(k=k.to(ty)) == mm3fa.ERR_DEVICE
    assert a(k=torch.zeros(2, 2, 30, 68, dtype=torch.uint8)) == mm3fa.ERR_DEVICE  # Q8_0
    assert a(k=torch.zeros(2, 2, 30, 64, dtype=torch.uint8)) == mm3fa.ERR_SHAPE
    assert a(v=k.bfloat16()) == mm3fa.ERR_TYPE
    assert a(q=q.double()) == mm3fa.ERR_TYPE
    assert a(q=q[:, :, :4]) == mm3fa.ERR_SHAPE   # not the tree's nodes
    assert a(q=q[:1]) == mm3fa.ERR_SHAPE         # not the slabs' sets
    assert a(q=q[:, :3]) == mm3fa.ERR_SHAPE      # heads that do not divide
    assert a(q=q[..., :32]) == mm3fa.ERR_SHAPE
    assert a(v=k[:, :, :29]) == mm3fa.ERR_SHAPE
    assert a(n=n[:1]) == mm3fa.ERR_SHAPE
    assert a(n=n.long()) == mm3fa.ERR_TYPE
    assert a(t=mm3fa.DraftTree(ints(3, 5))) == mm3fa.ERR_SHAPE  # 2 sequences are not a multiple of 3 trees
    assert a(scale=float("nan")) == mm3fa.ERR_SHAPE
    assert a(logit_softcap=-1.0) == mm3fa.ERR_SHAPE
    assert a(ws=WS[:1024]) == mm3fa.ERR_WORKSPACE
    assert a(ws=WS[4:]) == mm3fa.ERR_WORKSPACE  # 16-byte aligned
    out = torch.zeros(2, 5, 4, 64)
    assert a(out=out) == mm3fa.ERR_DEVICE
    assert a(out=out.half()) == mm3fa.ERR_TYPE
    assert a(q=q.half(), out=out) == mm3fa.ERR_DEVICE
    assert a(out=out.transpose(1, 2)) == mm3fa.ERR_SHAPE
    assert a(out=torch.zeros(2, 5, 1, 64).expand(2, 5, 4, 64)) == mm3fa.ERR_STRIDE
    for D in (32, 96, 512):
        assert a(q=torch.zeros(2, 4, 5, D), k=torch.zeros(2, 2, 30, D)) == mm3fa.ERR_UNSUPPORTED
    assert a(q=torch.zeros(2, 130, 5, 64)) == mm3fa.ERR_UNSUPPORTED  # 65 query heads for each kv head
    big = mm3fa.DraftTree(ints(1, 257))
    assert a(t=big, q=torch.zeros(2, 4, 257, 64)) == mm3fa.ERR_UNSUPPORTED
    assert big.attend_workspace(torch.zeros(2, 4, 257, 64), k, k) == 0
    assert t.attend_workspace(q, k, k) >= 1 << 16
    f, args = T_._calls()["attn"], (t._rows(q), T_._slab(k, t._dt, -1, ""), T_._slab(k, t._dt, -1, ""))
    end = (t._rows(out), WS.data_ptr(), WS.numel(), None)
    assert f(*args, None, n.data_ptr(), 0.1, 0.0, *end) == mm3fa.ERR_NULL
    assert f(*args, t._desc, None, 0.1, 0.0, *end) == mm3fa.ERR_NULL
    assert f(None, *args[1:], t._desc, n.data_ptr(), 0.1, 0.0, *end) == mm3fa.ERR_NULL
    assert f(*args, t._desc, n.data_ptr(), 0.1, 0.0, None, *end[1:]) == mm3fa.ERR_NULL
    for tree, want in (((8, 3, 0, 5, 2), mm3fa.ERR_SHAPE), ((8, 5, 0, 0, 1), mm3fa.ERR_SHAPE), ((6, 5, 0, 5, 1), mm3fa.ERR_ALIGN),
                       ((0, 5, 0, 5, 1), mm3fa.ERR_NULL), ((8, 0, 0, 5, 2), mm3fa.ERR_DEVICE)):
        assert f(*args, T_._PACK_TREE(*tree), n.data_ptr(), 0.1, 0.0, *end) == want


@no_gpu
def test_verify_refusals():
    t = mm3fa.DraftTree(ints(2, 5))
    lg, tok, acc, smp = torch.zeros(2, 5, 70), ints(2, 5), torch.zeros(2, 5), torch.zeros(2)
    a = lambda lg=lg, tok=tok, acc=acc, smp=smp, **kw: status(t.verify, lg, tok, acc, smp, **kw)
    assert a() == mm3fa.ERR_DEVICE
    for ty in (torch.float16, torch.bfloat16, torch.float32):
        assert a(lg=lg.to(ty), draft=lg.to(ty)) == mm3fa.ERR_DEVICE
    assert a(temperature=0.0) == mm3fa.ERR_DEVICE
    for temp in (-1.0, float("nan"), float("inf"), 1e-38):
        assert a(temperature=temp) == mm3fa.ERR_SHAPE
    assert a(lg=lg.double()) == mm3fa.ERR_TYPE
    assert a(lg=lg[0]) == mm3fa.ERR_SHAPE
    assert a(lg=lg[:, :4]) == mm3fa.ERR_SHAPE
    assert a(lg=lg[:1]) == mm3fa.ERR_SHAPE
    assert a(draft=lg[..., :69]) == mm3fa.ERR_SHAPE
    assert a(lg=lg[..., ::2]) == mm3fa.ERR_STRIDE
    assert a(tok=tok.long()) == mm3fa.ERR_TYPE
    assert a(tok=tok[:, :4]) == mm3fa.ERR_SHAPE
    assert a(tok=ints(5, 2).t()) == mm3fa.ERR_STRIDE
    assert a(acc=acc.half()) == mm3fa.ERR_TYPE
    assert a(smp=smp[:1]) == mm3fa.ERR_SHAPE
    assert a(smp=smp.half()) == mm3fa.ERR_TYPE
    assert a(smp=smp.double()) == mm3fa.ERR_TYPE
    assert a(out=(tok, ints(2), ints(1))) == mm3fa.ERR_SHAPE
    one = mm3fa.DraftTree(ints(1, 1))
    assert status(one.verify, torch.zeros(1, 1, 1).expand(1, 1, (1 << 22) + 1).clone(), ints(1, 1), torch.zeros(1, 1),
                  torch.zeros(1)) == mm3fa.ERR_UNSUPPORTED
    f = T_._calls()["verify"]
    good = [t._rows(lg[None]), None, t._desc, tok.data_ptr(), acc.data_ptr(), smp.data_ptr(), 1.0, tok.data_ptr(), tok.data_ptr(),
            tok.data_ptr(), None]
    assert f(*good) == mm3fa.ERR_DEVICE
    for i in (0, 2, 3, 4, 5, 7, 8, 9):
        assert f(*good[:i], None, *good[i + 1:]) == mm3fa.ERR_NULL
    for i in (3, 4, 5, 7, 8, 9):
        assert f(*good[:i], good[i] + 2, *good[i + 1:]) == mm3fa.ERR_ALIGN


@no_gpu
def test_commit_refusals():
    t = mm3fa.DraftTree(ints(1, 5))
    k = torch.zeros(3, 2, 2, 30, 64, dtype=torch.float16)
    path, n_path, n = ints(1, 5), ints(1), ints(2)
    C = mm3fa.CacheLayers
    a = lambda layers=None, path=path, n_path=n_path, n=n, **kw: status(t.commit, layers or C(k, k), path, n_path, n, **kw)
    assert a() == mm3fa.ERR_DEVICE
    for ty in (torch.bfloat16, torch.float32):
        assert a(C(k.to(ty), k.to(ty))) == mm3fa.ERR_DEVICE
    q8 = torch.zeros(3, 2, 2, 30, 68, dtype=torch.uint8)
    assert a(C(q8, q8)) == mm3fa.ERR_DEVICE
    assert status(C, k[:, 0], k[:, 0]) == mm3fa.ERR_SHAPE
    assert status(C, k, k[:2]) == mm3fa.ERR_SHAPE
    assert status(C, [], []) == mm3fa.ERR_SHAPE
    assert status(C, k.double(), k.double()) == mm3fa.ERR_TYPE
    assert status(C, k[..., ::2], k) == mm3fa.ERR_STRIDE
    assert status(C, q8[..., :67], q8) == mm3fa.ERR_SHAPE
    assert a(C(k, k.bfloat16())) == mm3fa.ERR_TYPE
    assert a(C(k, k[:, :, :, :29])) == mm3fa.ERR_SHAPE
    wide = torch.zeros(2, 2, 60, 64, dtype=torch.float16)[:, :, ::2]
    assert a(C([k[0], k[1], wide], k)) == mm3fa.ERR_STRIDE  # other strides than the first layer's
    assert a(C(k, [wide] * 3)) == mm3fa.ERR_DEVICE          # V's may be other ones than K's
    same = torch.zeros(1, 2, 30, 64, dtype=torch.float16).expand(2, 2, 30, 64)
    assert a(C([same], [same])) == mm3fa.ERR_STRIDE
    assert a(path=path[:, :4]) == mm3fa.ERR_SHAPE
    assert a(n_path=ints(2)) == mm3fa.ERR_SHAPE
    assert a(n=ints(3)) == mm3fa.ERR_SHAPE
    assert a(n=n.long()) == mm3fa.ERR_TYPE
    assert a(kv_len_out=n) == mm3fa.ERR_UNSUPPORTED
    t3 = mm3fa.DraftTree(ints(3, 5))
    assert status(t3.commit, C(k, k), ints(3, 5), ints(3), n) == mm3fa.ERR_SHAPE
    f, (kd, vd), m = T_._calls()["commit"], C(k, k)._desc, ints(2)
    good = [kd, vd, 3, path.data_ptr(), n_path.data_ptr(), 5, 1, n.data_ptr(), m.data_ptr(), None]
    assert f(*good) == mm3fa.ERR_DEVICE
    for i in (0, 1, 3, 4, 7, 8):
        assert f(*good[:i], None, *good[i + 1:]) == mm3fa.ERR_NULL
    for i in (2, 5, 6):
        assert f(*good[:i], 0, *good[i + 1:]) == mm3fa.ERR_SHAPE
    assert f(*good[:5], 257, *good[6:]) == mm3fa.ERR_UNSUPPORTED
    for i in (3, 4, 7, 8):
        assert f(*good[:i], good[i] + 2, *good[i + 1:]) == mm3fa.ERR_ALIGN
