"""What the header promises of the 8-bit paged cache's workspaces and sizes, on host tensors."""
import pytest
import torch

import kv8_ref
import mm3fa
from mm3fa import kv8

no_gpu = pytest.mark.skipif(torch.cuda.is_available(), reason="host tensors are accepted up to the device check only")


def make(**kw):
    kw = {"lens": [70, 5], "Hkv": 2, "D": 64, "P": 32, "room": [80, 40], **kw}
    return kv8_ref.State(**kw)


@pytest.mark.parametrize("n_pages,n_seq", [(1, 1), (512, 2), (100000, 65535)])
def test_a_workspace_holds_what_has_to_be_zeroed(n_pages, n_seq):
    """The first 64 KiB of a workspace are to be zeroed: it has as many bytes."""
    c = kv8._CACHE.pack(64, 32, 2, n_pages, 1, 0, *[1 << 20] * 4)
    f = kv8._calls()
    assert f["pages_workspace"](c, n_seq) >= 1 << 16
    assert f["pages_workspace"](c, n_seq) >= 4 * (3 * n_pages + 2 * n_seq)
    q = kv8._PACK_TENSOR(0, 0, 64, 1, 2, n_seq, 4, 256, 256, 512, 1 << 20)
    assert f["attn_workspace"](c, q, kv8._PACK_TABLE(1 << 20, 3, 3, n_seq)) >= 1 << 16
    bad = kv8._CACHE.pack(65, 32, 2, n_pages, 1, 0, *[1 << 20] * 4)
    assert f["pages_workspace"](bad, n_seq) == 0 and f["attn_workspace"](bad, q, kv8._PACK_TABLE(1 << 20, 3, 3, n_seq)) == 0


class Elsewhere:
    """A workspace on a device that the cache is not on."""
    device = "cuda:0"

    def __init__(self):
        self.t = torch.zeros(1 << 22, dtype=torch.uint8)

    def get_device(self):
        return 0

    def __getattr__(self, name):
        return getattr(self.t, name)


@no_gpu
def test_a_given_workspace_is_checked():
    """A workspace of another device, or one with gaps, is refused before its address goes anywhere."""
    s = make()
    c, q, out = s.cache(), torch.zeros(2, 4, 3, 64), torch.zeros(2, 3, 4, 64)
    with pytest.raises(ValueError):
        c.attend(0, q, s.table, s.len, 0.1, out, ws=Elsewhere())
    with pytest.raises(mm3fa.MM3FAError) as e:
        c.attend(0, q, s.table, s.len, 0.1, out, ws=torch.zeros(1 << 22, dtype=torch.uint8)[::2])
    assert e.value.status == mm3fa.ERR_STRIDE


@no_gpu
@pytest.mark.parametrize("P", [16, 32, 64, 128])
def test_a_table_whose_token_positions_leave_32_bits(P):
    """The attention rounds token counts up to its tiles in 32 bits: tables that near to 2^31 tokens are refused."""
    f, at = kv8._calls(), 1 << 20
    c = kv8._CACHE.pack(64, P, 1, 9, 1, 0, at, at, at, at)
    q = kv8._PACK_TENSOR(0, 0, 64, 1, 1, 1, 4, 256, 256, 256, at)
    for tokens, want in ((2 ** 31 - 8192, mm3fa.ERR_DEVICE), (2 ** 31 - 8192 + P, mm3fa.ERR_UNSUPPORTED), (2 ** 31 - P, mm3fa.ERR_UNSUPPORTED)):
        t = kv8._PACK_TABLE(at, tokens // P, tokens // P, 1)
        assert f["attn"](c, 0, q, t, at, None, 1.0, 0.0, 1, q, at, 1 << 40, None) == want
        assert (f["attn_workspace"](c, q, t) == 0) == (want == mm3fa.ERR_UNSUPPORTED)


@no_gpu
def test_a_given_workspace_of_page_operations_is_checked():
    s = make()
    c = s.cache()
    t2, l2, r2 = torch.empty_like(s.table), torch.empty_like(s.len), torch.empty_like(s.refs)
    one = torch.tensor([0], dtype=torch.int32)
    calls = (lambda ws: c.reserve(s.table, s.refs, s.len, ws=ws), lambda ws: c.compact(s.table, s.refs, t2, r2, ws=ws),
             lambda ws: c.fork(one, one, s.table, s.len, s.refs, t2, l2, r2, ws=ws),
             lambda ws: c.free(one, s.table, s.len, s.refs, t2, l2, r2, ws=ws))
    need = c.pages_workspace(2)
    for f in calls:
        for ws, want in ((torch.zeros(need, dtype=torch.uint8), mm3fa.ERR_DEVICE), (torch.zeros(need - 1, dtype=torch.uint8), mm3fa.ERR_WORKSPACE),
                         (torch.zeros(need + 8, dtype=torch.uint8)[2:], mm3fa.ERR_WORKSPACE),
                         (torch.zeros(2 * need, dtype=torch.uint8)[::2], mm3fa.ERR_STRIDE)):
            with pytest.raises(mm3fa.MM3FAError) as e:
                f(ws)
            assert e.value.status == want
        with pytest.raises(ValueError):
            f(Elsewhere())


@no_gpu
def test_no_capture_without_a_device():
    assert kv8._calls()["capture_id"](None) == 0
