"""The operators of decoding with a tree of drafted tokens: what is timed, in their plain form and through mm3fa.

A tree has T nodes; parents [n_tree, T] int32 names each node's parent, which comes before it (-1: none), node 0 is the
last accepted token; n_nodes [n_tree] says how many of them count.  Sequence s of N goes by tree s % n_tree, so that the
sets of a CFG pair share one.  The cache is a slab [N, Hkv, rows, D] of each layer; the nodes' K and V rows are behind
the kv_len tokens that a sequence holds, row kv_len + i being node i's.

  attend    softmax(scale * q k^T) v where a node sees the kv_len tokens, its ancestors and itself
  verify    which nodes stay: from node 0, the children of the accepted node in their order, each accepted with the
            target's probability over the draft's, else the target's left over by it; then the next token from what is
            left at the last accepted node.  Random numbers are inputs
  commit    the K and V rows of the accepted nodes moved behind the cache's, in all layers
"""
import torch

own = False  # set by the tools: run() makes mm3fa's calls instead of the plain form

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_Q8_BLOCK = 34  # bytes of 32 Q8_0 values


def _attend(name, N, trees, H, Hkv, D, T, width, kv_min, kv_max, dtype, cache, ragged=False):
    return {"name": name, "op": "attend", "N": N, "trees": trees, "H": H, "Hkv": Hkv, "D": D, "T": T, "width": width,
            "kv_min": kv_min, "kv_max": kv_max, "dtype": dtype, "cache": cache, "ragged": ragged}


def _verify(name, trees, T, width, V, dtype, draft, temperature, ragged=False):
    return {"name": name, "op": "verify", "trees": trees, "T": T, "width": width, "V": V, "dtype": dtype, "draft": draft,
            "temperature": temperature, "ragged": ragged}


def _commit(name, L, N, trees, Hkv, D, T, width, kv_min, kv_max, cache):
    return {"name": name, "op": "commit", "L": L, "N": N, "trees": trees, "Hkv": Hkv, "D": D, "T": T, "width": width,
            "kv_min": kv_min, "kv_max": kv_max, "cache": cache}


def listed():
    return [
        # the first steps of a song: a small tree of a CFG pair over a short prompt, where latency counts
        _attend("attend short pair", 2, 1, 32, 8, 128, 5, 2, 97, 311, "f32", "f16"),
        # a tree of a CFG pair at a long context, F32 activations as the graph has them
        _attend("attend pair 8192", 2, 1, 32, 8, 128, 24, 3, 8192, 8192, "f32", "f16"),
        # a server's batch of sequences of every length, each with a tree of its own
        _attend("attend ragged batch", 48, 48, 32, 8, 128, 13, 3, 1, 10240, "bf16", "bf16", True),
        # drafts in a row, without branches, small heads
        _attend("attend drafted rows", 7, 7, 16, 4, 64, 5, 1, 33, 2600, "f16", "f16", True),
        # a wide tree at a long context
        _attend("attend 64 nodes", 2, 1, 32, 8, 128, 64, 4, 8192, 8192, "bf16", "bf16"),
        # large trees of a few sequences
        _attend("attend 200 nodes", 8, 8, 32, 8, 128, 200, 3, 1900, 4100, "f16", "f16", True),
        # one small tree over a codebook's entries
        _verify("verify codebook", 1, 5, 2, 1025, "f32", "f32", 1.0),
        # a few trees whose drafts were drawn from a small model's distribution
        _verify("verify drawn drafts", 4, 24, 3, 32000, "bf16", "f32", 0.8),
        # a batch over a large vocabulary, the drafts being fixed choices
        _verify("verify large vocabulary", 64, 16, 2, 150001, "f32", "none", 1.0, True),
        # the pair's tree in all 36 layers
        _commit("commit pair", 36, 2, 1, 8, 128, 24, 3, 100, 900, "f16"),
        # a small model's Q8_0 cache
        _commit("commit q8_0", 4, 7, 7, 4, 64, 9, 2, 1, 300, "q8_0"),
        # a server's batch in all layers
        _commit("commit batch", 36, 48, 48, 8, 128, 13, 2, 20, 140, "bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "verify", "verify", "commit"])
    T = rng.choice([1, _log_int(rng, 2, 32), _log_int(rng, 2, 32), _log_int(rng, 33, 200)])
    width, trees = rng.choice([1, 2, 3, 4, 7]), _log_int(rng, 1, 48)
    Hkv, D = rng.choice([1, 2, 3, 4, 8]), rng.choice([64, 128, 128])
    if op == "verify":
        c = _verify("", _log_int(rng, 1, 64), T, width, _log_int(rng, 1000, 150000), rng.choice(["f32", "f16", "bf16"]),
                    rng.choice(["none", "f32", "bf16"]), round(rng.uniform(0.6, 1.2), 2), rng.random() < 0.5)
        while c["trees"] * c["T"] * c["V"] > 64 * 16 * 150001 // (1 if c["draft"] == "none" else 2):
            c["T"] = (c["T"] + 1) // 2
    elif op == "attend":
        cache = rng.choice(["f16", "bf16"])
        N = trees * rng.choice([1, 1, 2])
        kv_max = _log_int(rng, 2, 10240)
        c = _attend("", N, trees, Hkv * rng.choice([1, 2, 3, 4, 5, 8]), Hkv, D, T, width, _log_int(rng, 1, kv_max), kv_max,
                    rng.choice(["f32", cache]), cache, rng.random() < 0.5)
        most = work(listed()[2])["bytes"]
        while work(c)["bytes"] > most:
            c["kv_max"] = (c["kv_max"] + 1) // 2
            c["kv_min"] = min(c["kv_min"], c["kv_max"])
        most = work(listed()[5])["flops"]
        while work(c)["flops"] > most and c["T"] > 1:
            c["T"] = (c["T"] + 1) // 2
    else:
        L, sets = rng.choice([1, 4, 7, 36]), rng.choice([1, 1, 2])
        cache = rng.choice(["f16", "bf16", "f32", "q8_0"])
        kv_max = _log_int(rng, 2, 2000)
        while 2 * L * sets * trees * (kv_max + T) * Hkv * _row_bytes(cache, D) > 1100e6:
            kv_max, trees, T = (kv_max + 1) // 2, (trees + 1) // 2, (T + 1) // 2
        c = _commit("", L, sets * trees, trees, Hkv, D, T, width, 1, kv_max, cache)
    del c["name"]
    return c


def _lengths(lo, hi, N):
    """N lengths from lo to hi, evenly spread, both ends among them (the same for every seed)."""
    return [lo + (hi - lo) * ((i * 7) % N) // max(1, N - 1) for i in range(N)] if N > 1 else [hi]


def _row_bytes(cache, D):
    return D // 32 * _Q8_BLOCK if cache == "q8_0" else D * (4 if cache == "f32" else 2)


def _nodes(case):
    return _lengths(1, case["T"], case["trees"]) if case.get("ragged") else [case["T"]] * case["trees"]


def _parents(T, width):
    return [-1] + [(i - 1) // width for i in range(1, T)]


def _path(case, t):
    """The nodes of tree t that its inputs are made to accept: a branch, as deep as t says, within the tree's nodes."""
    T, w = _nodes(case)[t], case["width"]
    path, deep = [0], 1 + t % 5
    while len(path) <= deep and path[-1] * w + 1 < T:
        first = path[-1] * w + 1
        path.append(first + (t + len(path)) % min(w, T - first))
    return path


# ---------------------------------------------------------------- inputs

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def rand(*shape):
        return torch.rand(*shape, generator=g, device="cuda")

    def ints(x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")

    c, n_tree, T = dict(case), case["trees"], case["T"]
    s = {"case": c, "parents": ints([_parents(T, c["width"])] * n_tree), "n_nodes": ints(_nodes(c)) if c.get("ragged") else None}
    if c["op"] == "attend":
        N, H, Hkv, D, dt = c["N"], c["H"], c["Hkv"], c["D"], _TYPES[c["cache"]]
        held = _lengths(c["kv_min"], c["kv_max"], N)
        s["kv_len"] = ints(held)
        rows = max(held) + T
        s["k"], s["v"] = (torch.empty(N, Hkv, rows, D, dtype=dt, device="cuda") for _ in range(2))
        for i in range(N):
            s["k"][i] = randn(Hkv, rows, D)
            s["v"][i] = randn(Hkv, rows, D) * 0.5
        # q as the projection leaves it, [D, H, T, N], seen with the rows before the heads
        s["q"] = randn(N, T, H, D).to(_TYPES[c["dtype"]]).transpose(1, 2)
        s["out"] = torch.zeros(N, T, H, D, dtype=_TYPES[c["dtype"]], device="cuda")
    elif c["op"] == "verify":
        V, w = c["V"], c["width"]
        dt = _TYPES[c["dtype"]]
        s["logits"] = torch.empty(n_tree, T, V, dtype=dt, device="cuda")
        s["draft"] = None if c["draft"] == "none" else torch.empty(n_tree, T, V, dtype=_TYPES[c["draft"]], device="cuda")
        s["tokens"] = torch.zeros(n_tree, T, dtype=torch.int32, device="cuda")
        # numbers with 24 bits, below one; those of the nodes to be accepted are not the highest, the others' not the lowest
        s["accept"] = 0.5 + 0.5 * rand(n_tree, T)
        s["sample"] = rand(n_tree)
        par = torch.tensor(_parents(T, w), device="cuda")[1:]
        for t in range(n_tree):
            x = randn(T, V) * 2.0
            near = torch.softmax(0.7 * x + randn(T, V), -1)  # the small model's distribution, like the target's
            if T > 1:  # children drawn from their parent's row, or of the likeliest of it
                if s["draft"] is None:
                    rank = (torch.arange(1, T, device="cuda") - 1) % w
                    s["tokens"][t, 1:] = torch.topk(near, w, -1).indices[par, rank].to(torch.int32)
                else:
                    at = torch.cumsum(near, -1)
                    u = rand(T - 1, 1) * at[par, -1:]
                    s["tokens"][t, 1:] = torch.searchsorted(at[par], u).clamp(max=V - 1).view(-1).to(torch.int32)
                # the target thinks little of the drafts, but for those of the path
                x[par, s["tokens"][t, 1:].long()] -= 6.0
                path = _path(c, t)
                if len(path) > 1:
                    a, b = (torch.tensor(p, device="cuda") for p in (path[:-1], path[1:]))
                    x[a, s["tokens"][t, b].long()] = torch.logsumexp(x[a], -1) + 2.0
                    s["accept"][t, b] -= 0.5
            s["logits"][t] = x * c["temperature"]
            if s["draft"] is not None:
                s["draft"][t] = near
    else:
        L, N, Hkv, D = c["L"], c["N"], c["Hkv"], c["D"]
        held = _lengths(c["kv_min"], c["kv_max"], N)
        s["kv_len"], s["len_out"] = ints(held), ints(held)
        rows = max(held) + T
        if c["cache"] == "q8_0":
            shape = (L, N, Hkv, rows, _row_bytes("q8_0", D))
            s["k"], s["v"] = (torch.randint(0, 256, shape, generator=g, device="cuda", dtype=torch.uint8) for _ in range(2))
        else:
            s["k"], s["v"] = (torch.empty(L, N, Hkv, rows, D, dtype=_TYPES[c["cache"]], device="cuda") for _ in range(2))
            for l in range(L):
                s["k"][l] = randn(N, Hkv, rows, D)
                s["v"][l] = randn(N, Hkv, rows, D) * 0.5
        paths = [_path(c, t) for t in range(n_tree)]
        s["path"] = ints([p + [-1] * (T - len(p)) for p in paths])
        s["n_path"] = ints([len(p) for p in paths])
    return s


# ---------------------------------------------------------------- mm3fa's calls

def _mm3fa():
    import os
    import sys
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "minimaxmusic.cpp_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import mm3fa
    return mm3fa


def _own(s):
    c = s["case"]
    tree = s.get("tree")
    if tree is None:
        mm3fa = _mm3fa()
        tree = s["tree"] = mm3fa.DraftTree(s["parents"], s["n_nodes"])
        if c["op"] == "commit":
            s["layers"] = mm3fa.CacheLayers(s["k"], s["v"])
    if c["op"] == "attend":
        return tree.attend(s["q"], s["k"], s["v"], s["kv_len"], c["D"] ** -0.5, out=s["out"])
    if c["op"] == "verify":
        path, n_path, token = tree.verify(s["logits"], s["tokens"], s["accept"], s["sample"], draft=s["draft"],
                                          temperature=c["temperature"])
        return {"path": path, "n_path": n_path, "token": token}
    tree.commit(s["layers"], s["path"], s["n_path"], s["kv_len"], s["len_out"])
    return {"k": s["k"], "v": s["v"], "kv_len": s["len_out"]}


# ---------------------------------------------------------------- the plain form

def _ancestors(parents):
    """[n_tree, T, T]: whether node j is node i or one of its ancestors."""
    n, T = parents.shape
    eye = torch.eye(T, dtype=torch.bool, device=parents.device).expand(n, T, T)
    up = (parents[..., None] == torch.arange(T, device=parents.device)) | eye  # itself and its parent
    steps = 1
    while steps < T:  # twice as many steps up each time
        up = (up.float() @ up.float()) > 0
        steps *= 2
    return up


def _plain_attend(s):
    q, k, v, kv_len = s["q"], s["k"].float(), s["v"].float(), s["kv_len"]
    N, H, T, D = q.shape
    Hkv, rows = k.shape[1], k.shape[2]
    n_tree = s["parents"].shape[0]
    sc = (q.float().reshape(N, Hkv, H // Hkv * T, D) @ k.transpose(2, 3)) * D ** -0.5
    n_nodes = s["n_nodes"] if s["n_nodes"] is not None else torch.full((n_tree,), T, dtype=torch.int32, device=q.device)
    tree = torch.arange(N, device=q.device) % n_tree
    node = torch.arange(rows, device=q.device) - kv_len[:, None]  # [N, rows]: the node whose row it is, negative before
    of = node.clamp(0, T - 1)[:, None, :].expand(N, T, rows)
    seen = _ancestors(s["parents"])[tree].gather(2, of) & (node < T)[:, None]
    seen |= (node < 0)[:, None]
    sc = sc.view(N, H, T, rows).masked_fill_(~seen[:, None], float("-inf"))
    e = sc.sub_(sc.amax(-1, keepdim=True)).exp_()
    o = (e.view(N, Hkv, -1, rows) @ v).view(N, H, T, D) / e.sum(-1, keepdim=True)
    live = (torch.arange(T, device=q.device) < n_nodes[tree][:, None])[:, :, None, None]
    return torch.where(live, o.transpose(1, 2).to(s["out"].dtype), s["out"])


def _plain_verify(s):
    """In 64 bits: a decision is a comparison of computed numbers."""
    x, tokens, parents, draft = s["logits"], s["tokens"].long(), s["parents"], s["draft"]
    n, T, V = x.shape
    dev = x.device
    n_nodes = s["n_nodes"] if s["n_nodes"] is not None else torch.full((n,), T, dtype=torch.int32, device=dev)
    each = torch.arange(n, device=dev)

    def target(at):  # the target's probabilities behind node at[t] of each tree
        return torch.softmax(x[each, at].double() / s["case"]["temperature"], -1)

    cur = torch.zeros(n, dtype=torch.long, device=dev)
    left, mass = target(cur), torch.ones(n, dtype=torch.float64, device=dev)
    kept = torch.zeros(n, T, dtype=torch.bool, device=dev)
    kept[:, 0] = n_nodes > 0
    for i in range(1, T):  # children come after their parent: one pass over the nodes is the walk
        tested = (parents[:, i] == cur) & (i < n_nodes)
        tok = tokens[:, i]
        if draft is not None:
            q = draft[each, cur].double()
        else:
            q = torch.zeros_like(left).scatter_(1, tok[:, None], 1.0)
        ok = tested & (s["accept"][:, i].double() * q[each, tok] * mass < left[each, tok])
        no = tested & ~ok
        rest = (left - mass[:, None] * q).clamp_(min=0)
        kept[:, i] = ok
        cur = torch.where(ok, i, cur)
        left = torch.where(no[:, None], rest, torch.where(ok[:, None], target(cur), left))
        mass = torch.where(no, rest.sum(-1), torch.where(ok, 1.0, mass))
    left = torch.where((mass > 0)[:, None], left, target(cur))
    at = left.cumsum(-1)
    token = torch.searchsorted(at, (s["sample"].double() * at[:, -1])[:, None], right=True).view(-1).clamp(max=V - 1)
    node = torch.arange(T, device=dev)
    order = torch.where(kept, node, T).sort(-1).values
    return {"path": torch.where(order < T, order, -1).to(torch.int32), "n_path": kept.sum(-1).to(torch.int32),
            "token": torch.where(n_nodes > 0, token, -1).to(torch.int32)}


def _plain_commit(s):
    path, n_path, kv_len = s["path"], s["n_path"], s["kv_len"]
    N, T, rows = kv_len.shape[0], path.shape[1], s["k"].shape[3]
    tree = torch.arange(N, device=path.device) % path.shape[0]
    j = torch.arange(rows, device=path.device) - kv_len[:, None]  # place behind the cache's tokens
    moved = (j >= 0) & (j < n_path[tree][:, None])
    src = torch.where(moved, kv_len[:, None] + path[tree].gather(1, j.clamp(0, T - 1)), j + kv_len[:, None]).long()
    for x in ("k", "v"):
        L, _, Hkv, _, D = s[x].shape
        s[x].copy_(s[x].gather(3, src[None, :, None, :, None].expand(L, N, Hkv, rows, D)))
    s["len_out"].copy_(kv_len + n_path[tree])
    return {"k": s["k"], "v": s["v"], "kv_len": s["len_out"]}


_PLAIN = {"attend": _plain_attend, "verify": _plain_verify, "commit": _plain_commit}


def run(state):
    if own:
        return _own(state)
    return _PLAIN[state["case"]["op"]](state)


# ---------------------------------------------------------------- what it takes, and what is right

def _depths(T, width):
    d = [0]
    for i in range(1, T):
        d.append(d[(i - 1) // width] + 1)
    return d


def work(case):
    c, esz = case, {"f32": 4, "f16": 2, "bf16": 2, "none": 0}
    nodes, n_tree, deep = _nodes(c), c["trees"], _depths(c["T"], c["width"])
    if c["op"] == "attend":
        held = _lengths(c["kv_min"], c["kv_max"], c["N"])
        n = [nodes[s % n_tree] for s in range(c["N"])]
        pairs = sum(m * (h + 1) + sum(deep[:m]) for m, h in zip(n, held))
        cached = sum(h + m for m, h in zip(n, held)) * 2 * c["Hkv"] * c["D"] * esz[c["cache"]]
        return {"bytes": cached + 2 * sum(n) * c["H"] * c["D"] * esz[c["dtype"]], "flops": 4 * c["D"] * c["H"] * pairs}
    accepted = sum(len(_path(c, t)) for t in range(n_tree))
    if c["op"] == "verify":
        # the rows of the nodes on the path
        return {"bytes": accepted * c["V"] * (esz[c["dtype"]] + esz[c["draft"]]), "flops": 4 * accepted * c["V"]}
    moved = sum(len(_path(c, s % n_tree)) for s in range(c["N"]))
    return {"bytes": 4 * c["L"] * c["Hkv"] * moved * _row_bytes(c["cache"], c["D"]), "flops": 0}


def exact(case, seed):
    if case["op"] != "attend":
        return None  # whole numbers and copies: compared for equality
    s = prepare(case, seed)
    c = s["case"]
    D, group, n_tree, nodes, above = c["D"], c["H"] // c["Hkv"], c["trees"], _nodes(c), _parents(c["T"], c["width"])
    out = s["out"].double()
    for i, held in enumerate(s["kv_len"].tolist()):
        m = nodes[i % n_tree]
        shown = torch.zeros(m, held + m, dtype=torch.bool)
        shown[:, :held] = True
        for r in range(m):
            at = r
            while at >= 0:
                shown[r, held + at] = True
                at = above[at]
        hidden = torch.where(shown, 0.0, float("-inf")).double().to(s["q"].device)
        for h in range(c["Hkv"]):
            k, v = (s[x][i, h, :held + m].double() for x in ("k", "v"))
            a = torch.einsum("hrd,kd->hrk", s["q"][i, h * group:(h + 1) * group, :m].double(), k) / D ** 0.5 + hidden
            out[i, :m, h * group:(h + 1) * group] = torch.einsum("hrk,kd->rhd", torch.softmax(a, -1), v)
    return out
