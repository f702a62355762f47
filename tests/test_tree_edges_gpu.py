"""Tree decoding on the GPU where its ranges end, against the 64-bit references of tests/tree_ref.py."""
import random

import pytest
import torch

import mm3fa
import test_tree_gpu as base
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


def star_decisions(x, tokens, draft, temperature, turned_down):
    """F64 [n] each, for the child of the root behind `turned_down` ones that were turned down: its number u is accepted where
    u q M < r; and the sum c of the M before."""
    n = x.shape[0]
    each = torch.arange(n, device=x.device)
    r, mass = torch.softmax(x.double() / temperature, -1), torch.ones(n, dtype=torch.float64, device=x.device)
    c = torch.zeros_like(mass)
    for i in range(1, turned_down + 2):
        tok = tokens[:, i].long()
        q = torch.zeros_like(r).scatter_(1, tok[:, None], 1.0) if draft is None else draft.double()
        if i <= turned_down:
            r, c = (r - mass[:, None] * q).clamp(min=0), c + mass
            mass = r.sum(-1)
    return q[each, tok], mass, r[each, tok], c


@pytest.mark.parametrize("kind", ["likely", "dominant", "dominant twice", "rising", "drafts 0", "drafts 1", "drafts 3"])
@pytest.mark.parametrize("V", [300, 5003, 150001, (1 << 22) - 5])
def test_verify_decisions_next_to_their_border(cuda_device, V, kind):
    """Numbers two F32 steps below a decision's border accept, and two above it do not: a step is 2^-24 to 2^-23 of the number,
    F32 sums of the exponentials are off by more.  Children that had nearly all of the probability are turned down before."""
    n, temperature = 2 if V > 1 << 20 else 24, torch.tensor(0.7).item()  # as the call takes it, an F32 number: 0.7 itself moves p by 10^-7
    g = torch.Generator(device=cuda_device).manual_seed(V)
    x = torch.randn(n, V, generator=g, device=cuda_device) * 1.5
    if kind == "rising":
        x = x.sort(-1).values
    draft, down = None, {"likely": 1, "dominant": 1, "dominant twice": 2, "rising": 0}.get(kind, int(kind[-1]) if kind[-1].isdigit() else 0)
    tokens = torch.stack([torch.arange(n, device=cuda_device) * 7 % 50 + 51 * i for i in range(5)], 1).to(torch.int32)
    most = torch.logsumexp(x.double() / temperature, -1).float() * temperature
    if kind.startswith("dominant"):  # all but 2e-6 of the probability, and all but 5e-5 of the rest
        for i, more in ((1, 23.0 if down == 2 else 13.0), (2, 10.0))[:down]:
            x.scatter_(1, tokens[:, i:i + 1].long(), (most + more * temperature)[:, None])
    if kind == "likely":
        x.scatter_(1, tokens[:, 1:2].long(), most[:, None])
    if kind.startswith("drafts"):
        draft = torch.softmax(x / temperature + 0.3 * torch.randn(n, V, generator=g, device=cuda_device), -1)
        for i in range(1, down + 1):  # the draft thinks more of them than the target
            draft.scatter_(1, tokens[:, i:i + 1].long(), 1.5 * torch.softmax(x / temperature, -1).gather(1, tokens[:, i:i + 1].long()))
        _, mass, _, c = star_decisions(x, tokens, draft, temperature, down)
        p = torch.softmax(x / temperature, -1).gather(1, tokens[:, down + 1:down + 2].long())
        draft.scatter_(1, tokens[:, down + 1:down + 2].long(), p / (c + 0.5 * mass)[:, None].float())  # a border near 1/2
    q, mass, r, _ = star_decisions(x, tokens, draft, temperature, down)
    factor = q * mass
    border = (r / factor).float()
    assert ((border > 0) & (border < 0.999)).all()
    accept = torch.full((n, 5), 1.0 - 2.0 ** -24, device=cuda_device)
    T = down + 2
    logits = x[:, None].expand(n, T, V).contiguous()
    drafts = None if draft is None else draft[:, None].expand(n, T, V).contiguous()
    tree = mm3fa.DraftTree(torch.tensor([[-1] + [0] * (T - 1)], dtype=torch.int32, device=cuda_device).expand(n, T).contiguous())
    for way, taken in ((float("-inf"), True), (float("inf"), False)):
        u = border
        for _ in range(2):
            u = torch.nextafter(u, torch.full_like(u, way))
        accept[:, T - 1] = u
        assert ((u.double() * factor < r) == taken).all()
        path, n_path, token = tree.verify(logits, tokens[:, :T].contiguous(), accept[:, :T].contiguous(), torch.full((n,), 0.3, device=cuda_device),
                                          draft=drafts, temperature=temperature)
        assert ((n_path == 2) == taken).all() and (path[:, 1] == (T - 1 if taken else -1)).all(), (kind, taken)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("D,H,Hkv,T,lens", [(128, 8, 2, 5, [3, 250]), (64, 8, 2, 24, [1000, 63, 64, 65, 2500]), (128, 32, 8, 24, [4000, 3000]),
                                            (128, 16, 2, 70, [190, 191, 192, 193, 1200]), (64, 4, 4, 1, [0, 1, 127, 128])])
@pytest.mark.parametrize("cache", ["bf16", "f16"])
def test_attend_f32_results_keep_f32s_precision(cuda_device, D, H, Hkv, T, lens, dtype, cache):
    """The error of all rows together, as random as the inputs: of a weight, by the roundings of its exponent (four, of numbers
    around 7: 3.3e-7 by root mean square), 2^x (1.4e-7) and what the tensor core's sums of a score, whose last 8 additions are of
    its size, lose towards zero (3e-7); of a result, by those of its own (8 a tile: 4e-7).  Together 7e-7; 2^-19 allows for some
    2.5 times that.  (q and weights of 16 bits are off by 3.5e-6.)"""
    c = Case(cuda_device, lens, 1, H, Hkv, D, T, dtype, cache, seed=T + D)
    got = c.check(out=c.out(torch.float32))
    want, _ = R.attend(c.q, c.k, c.v, c.parents, None, c.len, c.scale, c.out(torch.float32))
    off = ((got.double() - want).norm() / want.norm()).item()
    assert off <= 2.0 ** -19, off


@pytest.mark.parametrize("dtype,cache", [("f32", "bf16"), ("bf16", "bf16"), ("f16", "bf16"), ("f32", "f16"), ("bf16", "f16"), ("f32", "f32")])
@pytest.mark.parametrize("D", [64, 128])
def test_attend_numbers_near_the_ends_of_f32(cuda_device, D, dtype, cache):
    """Queries, keys and values far from 1, with a scale that brings the scores back: the results are the same but for a power of two."""
    c = Case(cuda_device, [300, 5, 127], 1, 8, 2, D, 10, dtype, cache, seed=D + 1)
    out = c.out(torch.float32)
    q, k, v, scale = c.q, c.k, c.v, c.scale
    for up in (120, 90, -90, -118):
        if dtype != "f16":
            c.q = (q.float() * 2.0 ** up).to(q.dtype)
            c.check(out=out.clone(), scale=scale * 2.0 ** -up)
        c.q = q
        if cache != "f16":
            c.k = (k.float() * 2.0 ** up).to(k.dtype)
            c.check(out=out.clone(), scale=scale * 2.0 ** -up)
            c.k = k
            if up < 0:  # (rows far below the smallest numbers that results have are not asked for)
                continue
            c.v = (v.float() * 2.0 ** (up - 5)).to(v.dtype)
            c.check(out=out.clone())
            if dtype == cache:
                c.check(out=c.out())
            c.v = v


@pytest.mark.parametrize("dtype,cache", [("f32", "f16"), ("bf16", "bf16"), ("f32", "bf16")])
@pytest.mark.parametrize("N,H,Hkv,T,most", [(20, 32, 8, 40, 3000), (7, 48, 8, 100, 700), (90, 16, 2, 33, 400)])
def test_attend_groups_of_ctas_on_the_line(cuda_device, N, H, Hkv, T, most, dtype, cache):
    """More units than groups, of several CTAs each: every tree has all its nodes and more than 128 rows a kv head."""
    lens = [(i * 1237) % most for i in range(N)]
    Case(cuda_device, lens, 1, H, Hkv, 128, T, dtype, cache, seed=N).check()


@pytest.mark.parametrize("dtype,cache", [("f32", "f16"), ("bf16", "bf16"), ("f32", "bf16")])
@pytest.mark.parametrize("N,ratio,most,nodes", [(40, 4, 3000, None), (97, 8, 900, True), (140, 1, 2000, None), (33, 40, 1500, None)])
def test_attend_even_parts_of_many_sequences(cuda_device, N, ratio, most, nodes, dtype, cache):
    """Fewer units than CTAs, and more than 32 sequences: each lane of a planning warp has several."""
    T = 3
    lens = [(i * 1237) % most for i in range(N)]
    Case(cuda_device, lens, N if nodes else 1, ratio, 1, 128, T, dtype, cache, seed=N, n_nodes=[i % (T + 1) for i in range(N)] if nodes else None).check()


def far_apart(x, sets_apart):
    """x (2, Hkv, rows, ...) copied to memory whose second set begins more than 2^32 bytes behind the first."""
    big = torch.empty(sets_apart + x[0].numel(), dtype=x.dtype, device=x.device)
    view = big.as_strided(x.shape, (sets_apart, *x[0].contiguous().stride()))
    view.copy_(x)
    return view


@pytest.mark.parametrize("dtype,cache,odd", [("f32", "f32", 0), ("f32", "f16", 0), ("f32", "f16", 1), ("bf16", "bf16", 0)])
def test_attend_sets_more_than_4_gib_apart(cuda_device, dtype, cache, odd):
    """K and V of the second set behind 2^32 bytes, for the tensor-core kernel and the others (rows that are not aligned)."""
    c = Case(cuda_device, [300, 77], 1, 8, 2, 128, 6, dtype, cache, seed=20)
    apart = ((1 << 32) + (1 << 20)) // c.k.element_size() + odd
    c.k, c.v = far_apart(c.k, apart), far_apart(c.v, apart)
    assert c.k.stride(0) * c.k.element_size() > 1 << 32
    c.check()


def test_commit_and_verify_more_than_4_gib_apart(cuda_device):
    rng = random.Random(4)
    T, n = 20, 9
    k, v = (slabs(cuda_device, 2, 2, 2, 60, 64, "f16", seed) for seed in (1, 2))
    apart = ((1 << 32) + (1 << 20)) // 2
    far = [[far_apart(x, apart) for x in xs] for xs in (k, v)]
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda_device)
    path, lens = ints([rising(rng, T, n)]), ints([13, 38])
    want = [R.commit(xs, path, ints([n]), lens)[0] for xs in (k, v)]
    mm3fa.DraftTree(ints([[-1] * T])).commit(mm3fa.CacheLayers(*far), path, ints([n]), lens)
    assert all(torch.equal(a, b) for xs, ws in zip(far, want) for a, b in zip(xs, ws))

    def edit(s, par):
        s["logits"] = far_apart(s["logits"], ((1 << 32) + (1 << 20)) // 4)
    check_verify(cuda_device, 2, 12, 1025, "f32", None, 0.9, seed=3, edit=edit)


THREE = ("f32", "bf16")  # F32 results over BF16 slabs: three parts of q and weights, tiles of 64 keys


@pytest.mark.parametrize("T,H,Hkv,lens", [(40, 8, 2, [500, 0, 77, 260]), (128, 4, 1, [200, 31, 1, 129]), (256, 5, 1, [300, 2, 3, 4]), (67, 3, 3, [10, 400, 5, 6])])
def test_attend_large_trees_in_three_parts(cuda_device, T, H, Hkv, lens):
    base.test_attend_large_trees(cuda_device, T, H, Hkv, lens, *THREE)


def test_attend_what_is_seen_in_three_parts(cuda_device):
    """What is not seen, infinite values that are, in one of a CTA's units and between others, slabs' ends."""
    base.test_attend_what_is_not_seen_has_no_influence(cuda_device, *THREE)
    base.test_attend_infinite_values_that_are_seen(cuda_device, *THREE)
    base.test_attend_infinite_values_in_some_of_many(cuda_device, *THREE)
    c = Case(cuda_device, [128, 133, 140, 139], 1, 4, 2, 128, 9, *THREE, rows=140)
    c.len += torch.tensor([0, 0, 50, 0], dtype=torch.int32, device=cuda_device)
    c.check()
    for par in ([i - 1 for i in range(70)], [-1] + [0] * 69, [-1] * 70):
        Case(cuda_device, [90, 128], 1, 4, 2, 64, 70, *THREE, seed=3, parents=[par]).check()


@pytest.mark.parametrize("lens", [[(i * 37) % 100 for i in range(64)], [(i * 211) % 1500 for i in range(48)]])
def test_attend_many_pieces_in_three_parts(cuda_device, lens):
    """Units of one tile of 64 keys up to many, back to back and in a graph: no wait runs out, every result is the same."""
    base.test_attend_many_short_pieces(cuda_device, lens, *THREE)


@pytest.mark.parametrize("dtype,cache", [("f16", "bf16"), ("bf16", "f16")])
def test_attend_of_other_types_than_the_slabs(cuda_device, dtype, cache):
    base.test_attend_infinite_values_that_are_seen(cuda_device, dtype, cache)
    base.test_attend_what_is_not_seen_has_no_influence(cuda_device, dtype, cache)


@pytest.mark.parametrize("cache", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("up", [10, 17, 24])
def test_attend_small_elements_of_q_beside_a_large_one(cuda_device, up, cache):
    """One element of 2^up in each row of q, where the keys are 0.  Over F16 slabs the others are off by 2^-22 of themselves or
    2^-39 of the large one: a score by 2^(up - 39) |k| scale = 2^(up - 39) by root mean square, and the weights by as much;
    four times that on top of the bound for scores around 1."""
    c = Case(cuda_device, [300, 65], 1, 8, 2, 128, 10, "f32", cache, seed=up)
    c.k[..., 5] = 0
    c.q = c.q.clone()
    c.q[..., 5] = 2.0 ** up
    got = c.run()
    want, spread = R.attend(c.q, c.k, c.v, c.parents, None, c.len, c.scale, c.out())
    more = 4 * 2.0 ** (up - 39) if cache == "f16" else 0.0
    off = (got.double() - want).norm(dim=-1)
    assert (off <= (2.0 ** -17 + more) * spread + 2.0 ** -18 * want.norm(dim=-1)).all(), (off / want.norm(dim=-1)).max().item()


@pytest.mark.parametrize("dtype,cache", SIXTEEN + [("f32", "f32"), ("f32", "q8_0")])
@pytest.mark.parametrize("cap", [1e-38, 1e20, 1e31, 1e36, 3e38])
def test_attend_softcaps_from_the_smallest_to_the_largest(cuda_device, cap, dtype, cache):
    c = Case(cuda_device, [300, 5], 1, 8, 2, 128, 10, dtype, cache, seed=31)
    for scale in (c.scale, -c.scale, 1e-3 * c.scale):
        c.check(scale=scale, logit_softcap=torch.tensor(cap).item())


def test_commit_a_slab_of_one_head_as_k_and_v(cuda_device):
    """K of one layer is V of the next, under strides that differ along a dimension of one entry alone."""
    rng = random.Random(9)
    T, N = 24, 3
    some = slabs(cuda_device, 3, N, 1, T + 40, 64, "f16", 8)
    before = [x.clone() for x in some]
    other = lambda x: x.as_strided(x.shape, (x.stride(0), 8, x.stride(2), 1))
    path, n_path, lens = (torch.tensor(x, dtype=torch.int32, device=cuda_device) for x in ([rising(rng, T, 11)] * N, [11] * N, [0, 7, 33]))
    want, _ = R.commit(before, path, n_path, lens)
    layers = mm3fa.CacheLayers([some[0], some[1]], [other(some[2]), other(some[0])])
    mm3fa.DraftTree(torch.full((N, T), -1, dtype=torch.int32, device=cuda_device)).commit(layers, path, n_path, lens)
    assert all(torch.equal(x, w) for x, w in zip(some, want))
