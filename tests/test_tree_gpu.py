"""Decoding with a tree of drafted tokens on the GPU, against the 64-bit references of tests/tree_ref.py."""
import random

import pytest
import torch

import mm3fa
import tree_ref as R

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def random_parents(n_tree, T, seed, reach=4):
    rng = random.Random(seed)
    return [[-1] + [rng.randint(max(0, i - reach), i - 1) for i in range(1, T)] for _ in range(n_tree)]


def to_q8(x):
    """Q8_0 blocks (uint8) of a float tensor."""
    b = x.reshape(*x.shape[:-1], -1, 32)
    d = (b.abs().amax(-1, keepdim=True) / 127).half()
    c = (b / d.float().clamp(min=1e-8)).round().clamp(-127, 127).to(torch.int8)
    return torch.cat([d.view(torch.uint8), c.view(torch.uint8)], -1).reshape(*x.shape[:-1], -1)


class Case:
    """Slabs with `spare` rows behind the last node, random trees, queries seen with the rows before the heads."""

    def __init__(self, dev, lens, n_tree, H, Hkv, D, T, dtype="f16", cache="f16", seed=1, parents=None, n_nodes=None, spare=3, rows=None):
        g = torch.Generator(device=dev).manual_seed(seed)
        randn = lambda *s: torch.randn(*s, generator=g, device=dev)
        self.N, self.T, self.D = len(lens), T, D
        self.rows = rows or max(lens) + T + spare
        self.parents = torch.tensor(parents or random_parents(n_tree, T, seed), dtype=torch.int32, device=dev)
        self.n_nodes = None if n_nodes is None else torch.tensor(n_nodes, dtype=torch.int32, device=dev)
        self.len = torch.tensor(lens, dtype=torch.int32, device=dev)
        slab = lambda f: (lambda x: to_q8(x) if cache == R.Q8 else x.to(TYPES[cache]))(randn(self.N, Hkv, self.rows, D) * f)
        self.k, self.v = slab(1.0), slab(0.5)
        self.q = randn(self.N, T, H, D).to(TYPES[dtype]).transpose(1, 2)
        self.scale = D ** -0.5

    def tree(self):
        return mm3fa.DraftTree(self.parents, self.n_nodes)

    def out(self, dtype=None):
        return torch.full((self.N, self.T, self.q.shape[1], self.D), 7.0, dtype=dtype or self.q.dtype, device=self.q.device)

    def run(self, out=None, tree=None, **kw):
        return (tree or self.tree()).attend(self.q, self.k, self.v, self.len, kw.pop("scale", self.scale),
                                            out=self.out() if out is None else out, **kw)

    def check(self, got=None, **kw):
        tree = self.tree()
        got = self.run(tree=tree, **kw) if got is None else got
        want, spread = R.attend(self.q, self.k, self.v, self.parents, self.n_nodes, self.len, kw.get("scale", self.scale),
                                torch.full_like(got, 7.0), kw.get("logit_softcap", 0.0))
        R.check(got, want, spread, self.q, self.k)
        tree.check()
        return got


# ---------------------------------------------------------------- attention

@pytest.mark.parametrize("dtype,cache", [("f32", "f16"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "bf16"), ("f16", "bf16"), ("bf16", "f16"),
                                         ("f32", "f32"), ("bf16", "f32"), ("f32", "q8_0"), ("f16", "q8_0")])
@pytest.mark.parametrize("D,H,Hkv,T,lens", [(128, 8, 2, 5, [3, 250]), (64, 4, 4, 1, [0, 1, 130]), (128, 32, 2, 9, [127, 128, 129, 700]),
                                            (64, 6, 2, 33, [64, 95, 1]), (256, 4, 2, 7, [40, 300])])
def test_attend(cuda_device, D, H, Hkv, T, lens, dtype, cache):
    Case(cuda_device, lens, 1, H, Hkv, D, T, dtype, cache, seed=D + T).check()


@pytest.mark.parametrize("dtype,cache", [("f32", "f16"), ("f16", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("T,H,Hkv,lens", [(40, 8, 2, [500, 0, 77, 260]), (128, 4, 1, [200, 31, 1, 129]), (256, 5, 1, [300, 2, 3, 4]), (67, 3, 3, [10, 400, 5, 6]),
                                          (200, 16, 2, [1000, 90, 120, 130])])
def test_attend_large_trees(cuda_device, T, H, Hkv, lens, dtype, cache):
    """Several blocks of rows for each kv head, nodes over several tiles of keys, every second tree of its own size."""
    Case(cuda_device, lens, 2, H, Hkv, 128, T, dtype, cache, seed=T, n_nodes=[T, T // 2 + 1]).check()


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("parents", ["chain", "star", "forest", "invalid"])
def test_attend_shapes_of_trees(cuda_device, parents, dtype):
    T = 70
    par = {"chain": [i - 1 for i in range(T)], "star": [-1] + [0] * (T - 1), "forest": [-1] * T,
           "invalid": [3, -5, 2, 9, 1 << 30] + [-(1 << 31)] + [i for i in range(6, T)]}[parents]
    Case(cuda_device, [90, 128], 1, 4, 2, 128, T, dtype, seed=3, parents=[par]).check()


def test_attend_deep_trees(cuda_device):
    T = 256
    Case(cuda_device, [100, 129], 1, 2, 1, 64, T, seed=4, parents=[[i - 1 for i in range(T)]]).check()


@pytest.mark.parametrize("dtype,cache", [("f32", "f16"), ("bf16", "bf16")])
def test_attend_many_keys(cuda_device, dtype, cache):
    Case(cuda_device, [20011, 4095], 1, 4, 1, 128, 6, dtype, cache, seed=5).check()


@pytest.mark.parametrize("dtype,cache", [("f32", "f16"), ("bf16", "bf16"), ("f16", "f16")])
def test_attend_ragged_batch(cuda_device, dtype, cache):
    """Sequences of every length, some without nodes; two sets for each tree."""
    lens = [(i * 263) % 1500 for i in range(30)]
    Case(cuda_device, lens, 15, 8, 2, 128, 11, dtype, cache, seed=6, n_nodes=[(i * 5) % 13 - 1 for i in range(15)]).check()


def test_attend_rows_of_nodes_that_do_not_count(cuda_device):
    c = Case(cuda_device, [40, 300], 2, 8, 2, 128, 20, n_nodes=[0, 6])
    got = c.check()
    assert (got[0] == 7).all() and (got[1, 6:] == 7).all() and not (got[1, :6] == 7).any()
    made = c.tree().attend(c.q, c.k, c.v, c.len, c.scale)
    assert (made[0] == 0).all() and (made[1, 6:] == 0).all() and torch.equal(made[1, :6], got[1, :6])


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_attend_at_the_slabs_end(cuda_device, dtype):
    """Nodes whose rows lie behind the slab are absent; lengths are clamped to it; a node that sees nothing is zeros."""
    c = Case(cuda_device, [128, 133, 140, 139], 1, 4, 2, 128, 9, dtype, rows=140)
    c.len += torch.tensor([0, 0, 50, 0], dtype=torch.int32, device=cuda_device)
    c.check()
    c = Case(cuda_device, [0, -5 + 5], 1, 4, 2, 64, 9, dtype, rows=4, parents=[[-1] * 9])
    c.len[1] = -5
    got = c.check()
    assert (got[:, 4:] == 0).all()


def test_attend_strides(cuda_device):
    """Slabs and results that are parts of larger tensors, K and V of other strides, rows that are not 16-byte aligned."""
    for D, off, pad in ((128, 0, 64), (64, 8, 8), (128, 1, 3), (64, 2, 6)):
        c = Case(cuda_device, [200, 77], 1, 8, 2, D, 12, "f32", "f16", seed=7)
        big = torch.full((2, c.rows + 5, 2, D + pad), float("nan"), dtype=torch.float16, device=cuda_device)
        k = big[:, 2:2 + c.rows, :, off:off + D].transpose(1, 2)
        k.copy_(c.k)
        c.k = k
        qb = torch.full((2, 12, 9, D + pad), float("nan"), device=cuda_device)
        q = qb[:, :, 1:, off:off + D].transpose(1, 2)
        q.copy_(c.q)
        c.q = q
        ob = torch.full((2, 13, 9, D + pad), 7.0, device=cuda_device)
        out = ob[:, 1:, :8, off:off + D]
        c.check(c.run(out=out))
        assert (ob[:, 0] == 7).all() and (ob[:, :, 8] == 7).all() and (ob[..., :off] == 7).all() and (ob[..., off + D:] == 7).all()


def test_attend_after_a_refusal(cuda_device):
    """A refused call leaves nothing behind that a later one of the same shapes meets."""
    c = Case(cuda_device, [300, 150], 1, 8, 2, 64, 6, "f16", "f16", seed=9)
    tree, v = c.tree(), c.v
    for bad in (v.float(), v[:, :, :-1], v[:, :1]):
        c.v = bad
        with pytest.raises(mm3fa.MM3FAError):
            c.run(tree=tree)
    c.v = v
    c.check(c.run(tree=tree))
    tree.check()


def test_attend_strides_in_turn(cuda_device):
    """One tree with slabs of the same shape, first with rows that are not 16-byte aligned, then with aligned ones."""
    c = Case(cuda_device, [4000, 3000], 1, 8, 2, 128, 12, "f32", "f16", seed=8)
    tree, big = c.tree(), torch.zeros(2, 2, c.rows, 131, dtype=torch.float16, device=cuda_device)
    aligned, c.k = c.k, big[..., 1:129]
    c.k.copy_(aligned)
    need = tree.attend_workspace(c.q, c.k, c.v)
    c.check(c.run(tree=tree))
    c.k = aligned
    assert tree.attend_workspace(c.q, c.k, c.v) == need
    c.check(c.run(tree=tree))
    tree.check()


@pytest.mark.parametrize("dtype,cache", [("f32", "f16"), ("bf16", "bf16"), ("f32", "q8_0")])
def test_attend_scales_and_softcap(cuda_device, dtype, cache):
    c = Case(cuda_device, [300, 5], 1, 8, 2, 128, 10, dtype, cache, seed=8)
    for kw in ({"scale": -0.05}, {"scale": 0.0}, {"logit_softcap": 2.0}, {"scale": -0.08, "logit_softcap": 30.0}):
        c.check(**kw)


@pytest.mark.parametrize("dtype,cache", [("f32", "f16"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "bf16"), ("f32", "q8_0")])
def test_attend_what_is_not_seen_has_no_influence(cuda_device, dtype, cache):
    """NaN and infinities behind the nodes, in nodes that a node does not descend from, and in queries of others."""
    T, L = 40, 118
    c = Case(cuda_device, [L, 300], 1, 8, 2, 128, T, dtype, cache, seed=9, n_nodes=[T - 8], spare=40)
    want = c.run()
    dirty = lambda x, s, rows, value: x[s, :, rows].fill_(255) if x.dtype is torch.uint8 else x[s, :, rows].fill_(value)
    for value in (float("nan"), float("inf"), float("-inf")):
        k, v = c.k.clone(), c.v.clone()
        for s, n in ((0, L), (1, 300)):
            for x in (k, v):
                dirty(x, s, slice(n + T - 8, None), value)
        got = c.tree().attend(c.q, k, v, c.len, c.scale, out=c.out())
        assert torch.equal(got, want)
        if cache == "q8_0":
            continue
        bad = 11  # a node that few descend from
        for x in (k, v):
            x[0, 1, L + bad, 5] = value
            x[0, 0, L + bad] = value
        got = c.tree().attend(c.q, k, v, c.len, c.scale, out=c.out())
        sees = torch.tensor([bad in R.ancestors(c.parents[0].tolist(), i) for i in range(T)], device=cuda_device)
        assert torch.equal(got[1], want[1]) and torch.equal(got[0][~sees], want[0][~sees])
        assert not got[0][:T - 8][sees[:T - 8]].isfinite().all(-1).any()
    q = c.q.clone()
    q[0, 3, 4, 7], q[1, 0, 2, 1] = float("nan"), float("inf")
    got = c.tree().attend(q, c.k, c.v, c.len, c.scale, out=c.out())
    assert got[0, 4, 3].isnan().all() and got[1, 2, 0].isnan().all()
    got[0, 4, 3], got[1, 2, 0] = want[0, 4, 3], want[1, 2, 0]
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype,cache", [("f32", "f16"), ("f16", "f16"), ("bf16", "bf16")])
def test_attend_infinite_values_that_are_seen(cuda_device, dtype, cache):
    """An infinite element of a visible V row is an infinite element of the result, NaN where both signs meet."""
    T, L = 12, 200
    c = Case(cuda_device, [L], 1, 4, 2, 128, T, dtype, cache, seed=10, parents=[[-1, 0, 0, 1, 1, 2, 2, 3, 3, 4, 4, 5]])
    want = c.run()
    v, inf = c.v.clone(), float("inf")
    v[0, 0, L + 1, 3] = inf      # seen by 1 and below it
    v[0, 0, L + 3, 3] = -inf     # by 3, 7 and 8 too: NaN
    v[0, 0, 17, 9] = -inf        # by all
    got = c.tree().attend(c.q, c.k, v, c.len, c.scale, out=c.out())
    under = [[a in R.ancestors(c.parents[0].tolist(), i) for i in range(T)] for a in (1, 3)]
    for i in range(T):
        for h in (0, 1):  # the query heads of kv head 0
            assert got[0, i, h, 9] == -inf
            x = got[0, i, h, 3]
            assert x.isnan() if under[1][i] else (x == inf if under[0][i] else torch.equal(x, want[0, i, h, 3]))
    rest = torch.ones(128, dtype=torch.bool, device=cuda_device)
    rest[[3, 9]] = False
    assert torch.equal(got[..., rest], want[..., rest]) and torch.equal(got[:, :, 2:], want[:, :, 2:])


def test_attend_large_scores(cuda_device):
    """Scores of hundreds, among them the tile's last key, and rows whose first tile is far below the next."""
    c = Case(cuda_device, [300, 129], 1, 4, 2, 128, 8, "f32", "f16", seed=11)
    c.k[:, :, 250:260] *= 30
    c.k[:, :, 127] *= -40
    got = c.run()
    want, _ = R.attend(c.q, c.k, c.v, c.parents, None, c.len, c.scale, c.out())
    # scores reach 40 * 5: an F32 rounding of one, in log2 units and two parts of q, is 300 * 2^-21 of its weight
    err = ((got.double() - want).norm(dim=-1) / want.norm(dim=-1)).max().item()
    assert err <= 300 * 2.0 ** -20 * 2, err


def test_attend_long_slabs(cuda_device):
    """Offsets beyond 2^32 bytes: sets far apart in one large slab."""
    rows = 700000
    c = Case(cuda_device, [50, 60, 70], 1, 8, 4, 128, 6, "f32", "f16", seed=12)
    big = torch.zeros(3, 4, rows, 128, dtype=torch.float16, device=cuda_device)  # 2.1 GB
    far = torch.zeros(4, 4, rows, 128, dtype=torch.float16, device=cuda_device)
    assert far.numel() * 2 > 1 << 31 and far.stride(0) * 2 * 3 > 1 << 31
    big[:, :, :c.rows] = c.k
    far[1:, :, :c.rows] = c.v
    want = c.run()
    c.k, c.v = big, far[1:]
    assert torch.equal(c.run(), want)
    at = rows - 76  # and at the far end of the rows
    big[:, :, at:at + c.rows - 3] = big[:, :, :c.rows - 3].clone()
    far[1:, :, at:at + c.rows - 3] = far[1:, :, :c.rows - 3].clone()
    c.k, c.v = big[:, :, at:], far[1:, :, at:]
    assert torch.equal(c.run(), want)


def test_attend_is_the_same_every_time(cuda_device):
    for dtype, cache in (("f32", "f16"), ("bf16", "bf16")):
        c = Case(cuda_device, [5000, 300, 2999], 1, 16, 4, 128, 20, dtype, cache, seed=13)
        want = c.run()
        for _ in range(20):
            assert torch.equal(c.run(), want)


@pytest.mark.parametrize("dtype,cache", [("bf16", "bf16"), ("f32", "f16")])
@pytest.mark.parametrize("lens", [[(i * 37) % 100 for i in range(64)], [(i * 211) % 1500 for i in range(48)]])
def test_attend_many_short_pieces(cuda_device, lens, dtype, cache):
    """More units than SMs, of a tile or a few: every CTA goes from unit to unit, its warps at different places.  Back to
    back and in a graph, no wait runs out and every result is the same."""
    c = Case(cuda_device, lens, len(lens), 32, 8, 128, 13, dtype, cache, seed=16, n_nodes=[1 + i % 13 for i in range(len(lens))])
    tree = c.tree()
    want = c.check().clone()
    outs = [c.run(tree=tree) for _ in range(30)]
    tree.check()
    assert all(torch.equal(o, want) for o in outs)
    out = c.out()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        for _ in range(20):
            c.run(tree=tree, out=out)
    for _ in range(10):
        out.fill_(7.0)
        g.replay()
        torch.cuda.synchronize()
        tree.check(captured=True)
        assert torch.equal(out, want)


@pytest.mark.parametrize("dtype,cache", [("bf16", "bf16"), ("f32", "f16")])
def test_attend_infinite_values_in_some_of_many(cuda_device, dtype, cache):
    """Many units for every CTA, some with an infinite V element in a node's row: the units before and after them, of the same
    CTA, are as without it."""
    N, T = 120, 5
    c = Case(cuda_device, [(i * 29) % 90 for i in range(N)], 1, 8, 8, 64, T, dtype, cache, seed=18, parents=[[-1, 0, 0, 1, 1]])
    want = c.check().clone()
    v = c.v.clone()
    some = [i for i in range(N) if i % 5 in (1, 2)]
    for i in some:
        v[i, :, int(c.len[i]) + 1, 7] = float("inf")  # seen by nodes 1, 3 and 4
    tree = c.tree()
    for _ in range(5):
        got = tree.attend(c.q, c.k, v, c.len, c.scale, out=c.out())
        hit = torch.zeros_like(got, dtype=torch.bool)
        hit[torch.tensor(some)[:, None], torch.tensor([1, 3, 4]), :, 7] = True
        assert (got[hit] == float("inf")).all() and torch.equal(got[~hit], want[~hit])
    tree.check()


def test_attend_on_streams_and_in_graphs(cuda_device):
    """Two streams at once, a given stream, and two graphs replayed side by side with other lengths and trees."""
    c = Case(cuda_device, [3000, 1200], 1, 16, 4, 128, 20, "f32", "f16", seed=14)
    d = Case(cuda_device, [2500, 700], 1, 16, 4, 128, 20, "f32", "f16", seed=15)
    tree, want, other = c.tree(), c.run(), d.run()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    for s in (a, b):
        s.wait_stream(torch.cuda.current_stream())
    outs = [(c.run(tree=tree, stream=a), mm3fa.DraftTree(d.parents).attend(d.q, d.k, d.v, d.len, d.scale, stream=b)) for _ in range(10)]
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) and torch.equal(y, other) for x, y in outs)
    graphs = []
    for x in (c, d):
        out, t = x.out(), x.tree()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            for _ in range(3):
                x.run(out=out, tree=t)
        graphs.append((g, out, t))
    for _ in range(5):
        for s, (g, out, _) in zip((a, b), graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert torch.equal(graphs[0][1], want) and torch.equal(graphs[1][1], other)
    c.len -= 123
    c.parents.copy_(torch.tensor(random_parents(1, 20, 77), dtype=torch.int32))
    graphs[0][0].replay()
    torch.cuda.synchronize()
    c.check(graphs[0][1])
    for _, _, t in graphs:
        t.check(captured=True)


# ---------------------------------------------------------------- verification

def check_verify(dev, n_tree, T, V, dtype="f32", draft=None, temperature=1.0, seed=1, n_nodes=None, parents=None, edit=None, spread=1.5):
    g = torch.Generator(device=dev).manual_seed(seed)
    rand = lambda *s: torch.rand(*s, generator=g, device=dev)
    par = torch.tensor(parents or random_parents(n_tree, T, seed), dtype=torch.int32, device=dev)
    x = torch.randn(n_tree, T, V, generator=g, device=dev) * spread
    q = None if draft is None else torch.softmax(x + 0.5 * torch.randn(n_tree, T, V, generator=g, device=dev), -1).to(TYPES[draft])
    at = par.clamp(min=0).long()
    rows = torch.softmax(x, -1).gather(1, at[..., None].expand(-1, -1, V))
    tok = torch.multinomial(rows.view(-1, V), 1, generator=g).view(n_tree, T).to(torch.int32)
    s = {"logits": x.to(TYPES[dtype]), "tokens": tok, "accept": rand(n_tree, T), "sample": rand(n_tree), "draft": q}
    if edit:
        edit(s, par)
    nn = None if n_nodes is None else torch.tensor(n_nodes, dtype=torch.int32, device=dev)
    tree = mm3fa.DraftTree(par, nn)
    path, n_path, token = tree.verify(s["logits"], s["tokens"], s["accept"], s["sample"], draft=s["draft"], temperature=temperature)
    want = R.verify(s["logits"], s["tokens"], s["accept"], s["sample"], par, nn, s["draft"], temperature)
    for t, (p, w) in enumerate(want):
        assert int(n_path[t]) == len(p) and path[t].tolist() == p + [-1] * (T - len(p)), (t, p, path[t].tolist())
        assert int(token[t]) == w, (t, w, int(token[t]))
    return want


@pytest.mark.parametrize("draft", [None, "f32", "bf16", "f16"])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n_tree,T,V", [(3, 1, 2), (40, 9, 7), (17, 12, 255), (5, 20, 257), (9, 33, 5003), (2, 256, 600), (200, 5, 1025)])
def test_verify(cuda_device, n_tree, T, V, dtype, draft):
    want = check_verify(cuda_device, n_tree, T, V, dtype, draft, 0.9, seed=V + T, n_nodes=[(t * 7) % (T + 2) for t in range(n_tree)])
    # (a fixed choice is accepted with its probability, which is small here: test_verify_likely_choices)
    assert T < 9 or draft is None or any(len(p) > 1 for p, _ in want)


@pytest.mark.parametrize("n_tree,T,V", [(40, 12, 7), (9, 30, 1025), (3, 64, 40000)])
def test_verify_likely_choices(cuda_device, n_tree, T, V):
    """Fixed choices that the target thinks likely, siblings that repeat a token."""
    def edit(s, par):
        x, tok = s["logits"], s["tokens"]
        for t in range(n_tree):
            for i in range(1, T):
                x[t, par[t, i], tok[t, i]] = x[t, par[t, i]].logsumexp(-1) - 0.5 * (i % 3)
            tok[t, 2::5] = tok[t, 1:-1:5][:tok[t, 2::5].numel()]
    want = check_verify(cuda_device, n_tree, T, V, "f32", None, 1.0, seed=V, edit=edit)
    assert any(len(p) > 1 for p, _ in want)


@pytest.mark.parametrize("draft", [None, "f32"])
@pytest.mark.parametrize("n_tree,V", [(1, 150001), (3, 32000), (80, 20011)])
def test_verify_large_vocabularies(cuda_device, n_tree, V, draft):
    check_verify(cuda_device, n_tree, 6, V, "bf16" if draft else "f32", draft, 1.1, seed=V)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V", [1, 5, 3001, 70000])
def test_verify_greedy(cuda_device, V, dtype):
    """Temperature 0: the lowest of the tokens with the largest logit."""
    def edit(s, par):
        x = s["logits"]
        x[:, :, V // 2] = x[:, :, V // 3] = 9.0  # a tie
        x[1] = -1.0                              # and one of the whole vocabulary
        half = torch.rand(s["tokens"].shape, device=x.device) < 0.5
        s["tokens"][half] = V // 3
        s["tokens"][1] = 0
    want = check_verify(cuda_device, 6, 17, V, dtype, None, 0.0, seed=V, edit=edit)
    assert any(len(p) > 1 for p, _ in want) and all(w in (0, V // 3) for _, w in want)


@pytest.mark.parametrize("draft", [None, "f32"])
def test_verify_odd_inputs(cuda_device, draft):
    """Tokens outside the vocabulary and twice among the children of a node, logits of NaN, -inf and +inf, rows without any, random numbers at their ends, drafts of NaN and
    below zero, and drafts that are the target's own distribution, which leave nothing."""
    def edit(s, par):
        nan, inf = float("nan"), float("inf")
        x = s["logits"]
        s["tokens"][0, 1::2], s["tokens"][1, 2:] = 999, -1
        s["tokens"][2] = 5
        x[3, :, ::2] = -inf
        x[4, :, ::3] = nan
        x[5, 2:] = -inf
        x[6, :, 40] = x[6, :, 50] = inf
        s["tokens"][6, ::2] = 40
        x[7, 0] = -inf
        x[8, 0] = nan
        s["accept"][9:11], s["sample"][9], s["sample"][10] = 0.0, 0.0, 1.0 - 2.0 ** -24
        s["accept"][11], s["sample"][11], s["sample"][12] = nan, nan, 1.5
        s["sample"][13], s["accept"][14] = -3.0, 1.0
        x[15, :, 1:] = -inf  # one token has it all
        s["tokens"][15, ::2] = 0
        if s["draft"] is not None:
            s["draft"][16, :, ::2], s["draft"][16, :, 1::4] = nan, -1.0
            s["draft"][17] = inf
            s["draft"][18] = 0.0
    check_verify(cuda_device, 19, 24, 301, "f32", draft, 0.8, seed=21, edit=edit)


def test_verify_nothing_left(cuda_device):
    """Drafts that are exactly the target's distribution, all of them rejected: the next token is the target's."""
    V = 64
    x = torch.zeros(1, 4, V, device=cuda_device)
    q = torch.full((1, 4, V), 1.0 / V, device=cuda_device)
    tree = mm3fa.DraftTree(torch.tensor([[-1, 0, 0, 0]], dtype=torch.int32, device=cuda_device))
    tok = torch.tensor([[0, 3, 9, 9]], dtype=torch.int32, device=cuda_device)
    path, n_path, token = tree.verify(x, tok, torch.ones(1, 4, device=cuda_device), torch.full((1,), 0.51, device=cuda_device), draft=q)
    assert path.tolist() == [[0, -1, -1, -1]] and n_path.tolist() == [1] and token.tolist() == [int(0.51 * V)]


@pytest.mark.parametrize("draft", [None, "f32"])
def test_verify_tokens_follow_the_target(cuda_device, draft):
    """Over many trees the first token behind the root is distributed as the target has it, whatever the draft's is."""
    n, V, T = 60000, 6, 4
    g = torch.Generator(device=cuda_device).manual_seed(5)
    p = torch.tensor([0.4, 0.25, 0.2, 0.1, 0.05, 0.0], device=cuda_device)
    q = torch.tensor([0.1, 0.1, 0.1, 0.2, 0.2, 0.3], device=cuda_device)
    x = p.log().expand(n, T, V).contiguous()
    tree = mm3fa.DraftTree(torch.tensor([[-1, 0, 0, 0]], dtype=torch.int32, device=cuda_device).expand(n, T).contiguous())
    if draft is None:
        tok = torch.tensor([0, 3, 0, 5], dtype=torch.int32, device=cuda_device).expand(n, T).contiguous()
    else:
        tok = torch.multinomial(q.expand(n, V), T, replacement=True, generator=g).to(torch.int32)
    path, n_path, token = tree.verify(x, tok, torch.rand(n, T, generator=g, device=cuda_device), torch.rand(n, generator=g, device=cuda_device),
                                      draft=q.expand(n, T, V).contiguous() if draft else None)
    second = path[:, 1].long()
    first = torch.where(second > 0, tok.gather(1, second.clamp(min=0)[:, None]).view(-1), token)
    freq = torch.bincount(first.long(), minlength=V).double() / n
    sigma = (p.double() * (1 - p.double()) / n).sqrt()
    assert ((freq - p).abs() <= 5 * sigma + 1e-12).all(), freq


def test_verify_strides_and_streams(cuda_device):
    """Rows that are parts of larger ones, not aligned; a given stream; a captured call with new numbers."""
    n, T, V = 4, 10, 3001
    want = check_verify(cuda_device, n, T, V, "bf16", "f32", 1.0, seed=31)

    def edit(s, par):
        for name in ("logits", "draft"):
            big = torch.full((n, T + 1, V + 7), float("nan"), dtype=s[name].dtype, device=cuda_device)
            big[:, 1:, 3:3 + V] = s[name]
            s[name] = big[:, 1:, 3:3 + V]
    assert check_verify(cuda_device, n, T, V, "bf16", "f32", 1.0, seed=31, edit=edit) == want
    g = torch.Generator(device=cuda_device).manual_seed(1)
    tree = mm3fa.DraftTree(torch.tensor(random_parents(n, T, 1), dtype=torch.int32, device=cuda_device))
    x = torch.randn(n, T, V, generator=g, device=cuda_device)
    tok = x.argmax(-1).to(torch.int32).roll(1, 1)
    acc, smp = torch.rand(n, T, generator=g, device=cuda_device), torch.rand(n, generator=g, device=cuda_device)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    on_stream = tree.verify(x, tok, acc, smp, stream=s)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(on_stream, tree.verify(x, tok, acc, smp)))
    out = tuple(torch.empty_like(t) for t in on_stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tree.verify(x, tok, acc, smp, out=out)
    smp.copy_(1 - smp)
    acc.copy_(1 - acc)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(out, tree.verify(x, tok, acc, smp)))


# ---------------------------------------------------------------- commit

def slabs(dev, L, N, Hkv, rows, D, cache, seed=1):
    g = torch.Generator(device=dev).manual_seed(seed)
    b = {"f32": 4, "f16": 2, "bf16": 2}.get(cache)
    if cache == "q8_0":
        return [torch.randint(0, 256, (N, Hkv, rows, D // 32 * 34), generator=g, device=dev, dtype=torch.uint8) for _ in range(L)]
    return [torch.randn(N, Hkv, rows, D, generator=g, device=dev).to({4: torch.float32}.get(b, TYPES[cache])) for _ in range(L)]


def check_commit(dev, k, v, path, n_path, lens):
    path, n_path, lens = (torch.tensor(x, dtype=torch.int32, device=dev) for x in (path, n_path, lens))
    wk, wl = R.commit([x.clone() for x in k], path, n_path, lens)
    wv, _ = R.commit([x.clone() for x in v], path, n_path, lens)
    tree = mm3fa.DraftTree(torch.full(path.shape, -1, dtype=torch.int32, device=dev))
    got = tree.commit(mm3fa.CacheLayers(k, v), path, n_path, lens)
    assert torch.equal(got, wl), (got, wl)
    same = lambda a, b: torch.equal(a.view(torch.uint8) if a.is_contiguous() else a, b.view(torch.uint8) if a.is_contiguous() else b)
    assert all(same(a, b) for a, b in zip(k, wk)) and all(same(a, b) for a, b in zip(v, wv))
    return got


def rising(rng, T, n):
    return [0] + sorted(rng.sample(range(1, T), n - 1)) + [-1] * (T - n)


@pytest.mark.parametrize("cache", ["f16", "bf16", "f32", "q8_0"])
@pytest.mark.parametrize("L,N,n_tree,Hkv,D,T", [(1, 1, 1, 1, 64, 1), (3, 4, 2, 2, 128, 24), (36, 2, 1, 8, 128, 9), (2, 3, 3, 3, 256, 200), (100, 2, 2, 1, 64, 40),
                                                (2, 2, 1, 2, 96, 256)])
def test_commit(cuda_device, L, N, n_tree, Hkv, D, T, cache):
    rng = random.Random(T)
    counts = [max(1, T - 3 * t) if t % 2 else max(1, T // 3) for t in range(n_tree)]
    k, v = (slabs(cuda_device, L, N, Hkv, T + 60, D, cache, seed) for seed in (1, 2))
    check_commit(cuda_device, k, v, [rising(rng, T, n) for n in counts], counts, [rng.randint(0, 60) for _ in range(N)])


@pytest.mark.parametrize("L,N,Hkv", [(37, 64, 8), (97, 65, 5), (13, 1200, 8)])
def test_commit_many_sets_and_layers(cuda_device, L, N, Hkv):
    """More sets, heads and layers than there are warps: some take one layer more than others."""
    rng = random.Random(L)
    counts = [1 + i % 5 for i in range(N)]
    k, v = (slabs(cuda_device, L, N, Hkv, 20, 64, "f16", seed) for seed in (5, 6))
    check_commit(cuda_device, k, v, [rising(rng, 9, n) for n in counts], counts, [rng.randint(0, 12) for _ in range(N)])


def test_commit_paths_that_end_early(cuda_device):
    k, v = (slabs(cuda_device, 2, 9, 2, 50, 64, "f16", seed) for seed in (3, 4))
    T = 40
    pad = lambda p: p + [-1] * (T - len(p))
    paths = [pad([0, 2, 2, 5]), pad([0, 3, 1]), pad([2, 5, 60]), pad([-1, 3]), pad([0, 7, 9]), pad([0, 2, 4]), pad([]),
             list(range(0, T)), pad([0] + list(range(5, 40)))]
    got = check_commit(cuda_device, k, v, paths, [4, 3, 3, 2, -2, 99, 3, 40, 36], [1, 2, 3, 4, 5, 6, -7, 20, 30])
    assert got.tolist() == [3, 4, 5, 4, 5, 9, -7, 50, 46]


def test_commit_strided_slabs(cuda_device):
    """Views of a larger cache, with rows that allow accesses of 2, 4, 8 and 16 bytes; what is between them stays."""
    rng = random.Random(1)
    for off, wide in ((0, 128), (1, 67), (2, 70), (4, 72)):
        base = [torch.randn(2, 40, 3, wide, device=cuda_device).half() for _ in range(4)]
        before = [b.clone() for b in base]
        views = lambda bs: [b[:, 2:, 1:, off:off + 64].transpose(1, 2) for b in bs]
        k, v = views(base[:2]), views(base[2:])
        path = [rising(rng, 12, 7)]
        wk, _ = R.commit(views(before), torch.tensor(path), [7], torch.tensor([5, 20]))
        tree = mm3fa.DraftTree(torch.zeros(1, 12, dtype=torch.int32, device=cuda_device))
        ints = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda_device)
        tree.commit(mm3fa.CacheLayers(k, v), ints(path), ints([7]), ints([5, 20]))
        for b, old, w in zip(base, before, wk):
            old[:, 2:, 1:, off:off + 64].transpose(1, 2).copy_(w)
            assert torch.equal(b, old)


# ---------------------------------------------------------------- together

def test_tree_decoding_gives_the_tokens_of_single_steps(cuda_device):
    """A small random model, two sets of a CFG pair: greedy decoding with trees, some branches of which are right, gives
    the tokens that one token a step gives.  Prologue, attention, verification and commit, all through one cache."""
    from mm3fa import ggml

    dev, D, H, Hkv, layers, V, rows, N = cuda_device, 64, 4, 2, 2, 97, 96, 2
    g = torch.Generator(device=dev).manual_seed(3)
    w = lambda *s: torch.randn(*s, generator=g, device=dev) / s[-1] ** 0.5
    E = H * D
    emb = torch.randn(N, V, E, generator=g, device=dev)  # the sets see the same tokens, differently
    W = [(w(H * D, E), w(Hkv * D, E), w(Hkv * D, E), w(E, H * D)) for _ in range(layers)]
    head = w(V, E) * 4
    norm = torch.ones(D, device=dev)

    def prologue(x, wq, wk, wv, kc, vc, pos, tok_rows):
        """[N, T, E] -> q [N, T, H, D]; K and V rows of every node stored (one set for each node, of a slab with all rows)."""
        T = x.shape[1]
        q, k, v = (torch.nn.functional.linear(x, m).reshape(N * T, -1, D).contiguous() for m in (wq, wk, wv))
        q_out = torch.empty_like(q)
        d3 = lambda t: ggml.make(ggml.GGML_TYPE_F32, [D, t.shape[1], N * T], t.data_ptr())
        slab = lambda c: ggml.make(ggml.GGML_TYPE_F16, [D, N * Hkv * rows, Hkv, N * T], c.data_ptr(), [2, 2 * D, 2 * D * rows, 0])
        at = (tok_rows + torch.arange(N, device=dev)[:, None] * Hkv * rows).reshape(-1).long().contiguous()
        pos = pos.reshape(-1).to(torch.int32).contiguous()
        mm3fa.decode_prologue(d3(q), d3(k), d3(v), norm.data_ptr(), norm.data_ptr(), 1e-6, pos.data_ptr(), 1e4, at.data_ptr(), slab(kc), slab(vc),
                              d3(q_out), torch.cuda.current_stream().cuda_stream)
        return q_out.view(N, T, H, D)

    def forward(tree, parents, tokens, kv_len, kc, vc):
        """Logits [T, V] of a tree's nodes behind kv_len tokens."""
        T = len(parents)
        depth = [0]
        for i in range(1, T):
            depth.append(depth[parents[i]] + 1)
        depth = torch.tensor(depth, device=dev)
        x = emb[:, tokens]
        for l, (wq, wk, wv, wo) in enumerate(W):
            q = prologue(x, wq, wk, wv, kc[l], vc[l], kv_len[:, None] + depth, kv_len[:, None] + torch.arange(T, device=dev))
            o = tree.attend(q.transpose(1, 2), kc[l], vc[l], kv_len, D ** -0.5)
            x = x + torch.nn.functional.linear(o.reshape(N, T, H * D), wo)
        cond, uncond = torch.nn.functional.linear(x, head)
        return uncond + 1.5 * (cond - uncond)

    def decode(n_tokens, drafts):
        """Greedy tokens; drafts(step): (parents, tokens of the nodes behind the root)."""
        kc, vc = (torch.zeros(layers, N, Hkv, rows, D, dtype=torch.float16, device=dev) for _ in range(2))
        cache = mm3fa.CacheLayers(kc, vc)
        kv_len = torch.zeros(N, dtype=torch.int32, device=dev)
        out, margin, steps = [5], 1e9, 0
        while len(out) < n_tokens:
            parents, rest = drafts(out)
            tree = mm3fa.DraftTree(torch.tensor([parents], dtype=torch.int32, device=dev))
            tokens = torch.tensor([[out[-1]] + rest], dtype=torch.int32, device=dev)
            logits = forward(tree, parents, tokens[0].long(), kv_len, kc, vc)
            zeros = torch.zeros(1, len(parents), device=dev)
            path, n_path, token = tree.verify(logits[None].contiguous(), tokens, zeros, zeros[:, 0].contiguous(), temperature=0.0)
            kv_len = tree.commit(cache, path, n_path, kv_len)
            kept = path[0, :int(n_path)].long()
            two = logits[kept].topk(2, -1).values
            margin = min(margin, float((two[:, 0] - two[:, 1]).min()))
            out += tokens[0, kept[1:]].tolist() + [int(token)]
            tree.check()
            steps += 1
        return out[:n_tokens], margin, steps

    single, margin, steps = decode(60, lambda out: ([-1], []))
    assert steps == 59 and margin > 1e-3  # (an F32 sum taken otherwise moves a logit of 10 by 1e-5)
    rng = random.Random(2)

    def branches(out):
        """A chain of the right tokens, broken at times, beside wrong ones."""
        n, parents, tokens, at = len(out), [-1], [], 0
        for d in range(rng.randint(0, 4)):
            wrong = [rng.randrange(V) for _ in range(rng.randint(0, 2))]
            right = single[n + d] if n + d < len(single) and rng.random() < 0.8 else rng.randrange(V)
            kids = wrong + [right]
            first = len(parents)
            parents += [at] * len(kids)
            tokens += kids
            at = first + len(kids) - 1
        return parents, tokens

    got, _, steps = decode(60, branches)
    assert got == single and steps < 45
