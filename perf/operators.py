"""The operators of the 8-bit paged KV cache: what is timed, in their plain form and through mm3fa.

The cache holds K and V of L layers as 8-bit codes in pages of P tokens, with one F32 scale for each
page and kv head (value = code * scale):

  k, v               int8 [L, n_pages, n_head_kv, P, D]
  k_scale, v_scale   F32  [L, n_pages, n_head_kv]
  table              int32 [N, max_pages]: page of tokens [P*j, P*j + P) of sequence s, -1 where there is none
  kv_len             int32 [N]: tokens of each sequence that the cache holds
  refs               int32 [n_pages]: how many table entries name each page (0: free)

  attend    softmax(scale * q k^T) v over each sequence's pages, causal at its end, rows past q_len left as they were
  append    new K and V rows into the pages: the scale of a page grows to max|x| / 127 over its new rows and the
            codes that it held are rounded to the new scale; read: the rows' values back out of the pages
  fork      sequences take over the pages of others (shared, the partly filled last page copied; or all of them copied)
  compact   the live pages moved to the front of the pool
"""
import torch

own = False  # set by the tools: run() makes mm3fa's calls instead of the plain form

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _attend(name, N, H, Hkv, D, P, n_q, kv_min, kv_max, dtype, ragged_q=False):
    return {"name": name, "op": "attend", "N": N, "H": H, "Hkv": Hkv, "D": D, "P": P, "n_q": n_q, "kv_min": kv_min,
            "kv_max": kv_max, "dtype": dtype, "ragged_q": ragged_q}


def _append(name, N, Hkv, D, P, T, start_min, start_max, dtype):
    return {"name": name, "op": "append", "N": N, "Hkv": Hkv, "D": D, "P": P, "T": T, "start_min": start_min,
            "start_max": start_max, "dtype": dtype}


def _fork(name, L, N, Hkv, D, P, kv_min, kv_max, pairs, deep):
    return {"name": name, "op": "fork", "L": L, "N": N, "Hkv": Hkv, "D": D, "P": P, "kv_min": kv_min, "kv_max": kv_max,
            "pairs": pairs, "deep": deep}


def _compact(name, L, N, Hkv, D, P, kv_min, kv_max, holes):
    return {"name": name, "op": "compact", "L": L, "N": N, "Hkv": Hkv, "D": D, "P": P, "kv_min": kv_min,
            "kv_max": kv_max, "holes": holes}


def listed():
    return [
        # the first steps of a song: one token of a CFG pair over a short prompt, where latency counts
        _attend("attend short pair", 2, 32, 8, 128, 64, 1, 97, 311, "f32"),
        # the decode step at a long context: one token of a CFG pair, F32 activations as the graph has them
        _attend("attend pair 8192", 2, 32, 8, 128, 64, 1, 8192, 8192, "f32"),
        # a server's batch of sequences of every length
        _attend("attend ragged batch", 48, 32, 8, 128, 64, 1, 1, 10240, "bf16"),
        # a few drafted tokens for each sequence, small heads, small pages
        _attend("attend drafted rows", 7, 16, 4, 64, 16, 5, 33, 2600, "f16"),
        # a prompt's prefill, both sets of the CFG pair, F32 activations
        _attend("attend prefill 1024", 2, 32, 8, 128, 64, 1024, 1024, 1024, "f32"),
        # a chunk of a long prompt after what the cache holds of it
        _attend("attend chunk of 2048", 1, 32, 8, 128, 64, 2048, 8192, 8192, "bf16"),
        # the decode step's new row of each set
        _append("append one token", 2, 8, 128, 64, 1, 100, 8191, "f32"),
        # a prompt's rows, starting inside a page
        _append("append prompt", 2, 8, 128, 64, 4096, 0, 63, "f32"),
        # candidates of one prompt: full pages shared, the last one copied, in a small model
        _fork("fork shared", 4, 16, 2, 64, 16, 1, 700, 7, False),
        # independent copies of long sequences, all 36 layers
        _fork("fork deep", 36, 8, 8, 128, 64, 900, 2500, 3, True),
        # a small pool after a few sequences have ended
        _compact("compact small", 4, 16, 2, 64, 16, 1, 300, 0.3),
        # a full-sized pool, half of it free in pieces
        _compact("compact 36 layers", 36, 8, 8, 128, 64, 300, 1200, 0.5),
    ]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "append", "fork", "compact"])
    D, P = rng.choice([64, 128, 128, 256]), rng.choice([16, 32, 64, 128])
    Hkv = rng.choice([1, 2, 3, 4, 8])
    if op == "attend":
        H, N = Hkv * rng.choice([1, 2, 3, 4, 5, 8]), _log_int(rng, 1, 48)
        kv_max = _log_int(rng, 2, 10240)
        n_q = rng.choice([1, 1, 1, _log_int(rng, 2, 16), _log_int(rng, 17, 1100)])
        n_q = min(n_q, kv_max)
        c = _attend("", N, H, Hkv, D, P, n_q, _log_int(rng, n_q, kv_max), kv_max, rng.choice(["f32", "f16", "bf16"]),
                    n_q > 1 and rng.random() < 0.5)
        limit = work(listed()[5])["flops"]
        while work(c)["flops"] > limit and c["N"] > 1:
            c["N"] = (c["N"] + 1) // 2
        while work(c)["flops"] > limit:
            c["n_q"] = (c["n_q"] + 1) // 2
    elif op == "append":
        N, T = _log_int(rng, 1, 48), rng.choice([1, _log_int(rng, 2, 4096)])
        c = _append("", N, Hkv, D, P, T, 0, _log_int(rng, 1, 8191), rng.choice(["f32", "f16", "bf16"]))
        limit = work(listed()[7])["bytes"]
        while work(c)["bytes"] > limit and c["T"] > 1:
            c["T"] = (c["T"] + 1) // 2
    else:
        L, N, kv_max = rng.choice([1, 4, 7, 36]), _log_int(rng, 2, 64), _log_int(rng, 2, 2500)
        while 2 * L * N * kv_max * Hkv * D > 600e6 and N > 2:
            N = (N + 1) // 2
        while 2 * L * N * kv_max * Hkv * D > 600e6:
            kv_max = (kv_max + 1) // 2
        if op == "fork":
            c = _fork("", L, N, Hkv, D, P, 1, kv_max, rng.randint(1, N - 1), rng.random() < 0.5)
        else:
            c = _compact("", L, N, Hkv, D, P, 1, kv_max, round(rng.uniform(0.1, 0.8), 2))
    del c["name"]
    return c


def _lengths(lo, hi, N):
    """N lengths from lo to hi, evenly spread, both ends among them (the same for every seed)."""
    return [lo + (hi - lo) * ((i * 7) % N) // max(1, N - 1) for i in range(N)] if N > 1 else [hi]


def _pages(n, P):
    return -(-n // P)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def randperm(n):
        return torch.randperm(n, generator=g, device="cuda")

    c, op = dict(case), case["op"]
    N, Hkv, D, P, L = c["N"], c["Hkv"], c["D"], c["P"], c.get("L", 1)
    if op == "append":
        held = _lengths(c["start_min"], c["start_max"], N)
        room = [h + c["T"] for h in held]
    else:
        held = room = _lengths(c["kv_min"], c["kv_max"], N)
    used = [_pages(n, P) for n in room]
    total = sum(used)
    if op == "fork":
        n_pages = 2 * total + c["pairs"] * max(used) + 3
    elif op == "compact":
        n_pages = int(total / (1 - c["holes"])) + 1
    else:
        n_pages = total + 3
    # codes as a scale of max/127 over a page of normal values leaves them, scales around 4/127
    def pool():
        x = torch.empty(L, n_pages, Hkv, P, D, dtype=torch.int8, device="cuda")
        for l in range(L):
            x[l] = (randn(n_pages, Hkv, P, D) * 32).round().clamp(-127, 127).to(torch.int8)
        return x

    s = {"case": c, "k": pool(), "v": pool()}
    s["k_scale"] = 0.031 * torch.exp(0.2 * randn(L, n_pages, Hkv))
    s["v_scale"] = 0.016 * torch.exp(0.5 * randn(L, n_pages, Hkv))
    # every sequence's pages, scattered over the pool
    order = randperm(n_pages)[:total].to(torch.int32)
    table = torch.full((N, max(used) + 1), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(used):
        table[i, :n] = order[at:at + n]
        at += n
    s["table"] = table
    s["kv_len"] = torch.tensor(held, dtype=torch.int32, device="cuda")
    if op == "attend":
        dt = _TYPES[c["dtype"]]
        # q as the projection leaves it, [D, H, n_q, N], seen with the rows before the heads
        s["q"] = randn(N, c["n_q"], c["H"], D).to(dt).transpose(1, 2)
        s["out"] = torch.zeros(N, c["n_q"], c["H"], D, dtype=dt, device="cuda")
        s["q_len"] = None
        if c["ragged_q"]:
            s["q_len"] = torch.tensor([min(n, h) for n, h in zip(_lengths(1, c["n_q"], N), held)], dtype=torch.int32, device="cuda")
    elif op == "append":
        dt = _TYPES[c["dtype"]]
        s["k_new"] = randn(N, c["T"], Hkv, D).to(dt).transpose(1, 2)
        s["v_new"] = (randn(N, c["T"], Hkv, D) * 0.5).to(dt).transpose(1, 2)
        # read back from the first page that is written on, the rows that it held among them
        s["first"] = s["kv_len"] // P * P
        s["rows"] = s["kv_len"] - s["first"] + c["T"]
        s["k_out"] = torch.zeros(N, Hkv, c["T"] + P - 1, D, device="cuda")
        s["v_out"] = torch.zeros(N, Hkv, c["T"] + P - 1, D, device="cuda")
    else:
        s["refs"] = torch.zeros(n_pages, dtype=torch.int32, device="cuda")
        s["refs"][order.long()] = 1
        s["table_out"], s["refs_out"], s["kv_len_out"] = torch.empty_like(table), torch.empty_like(s["refs"]), torch.empty_like(s["kv_len"])
        if op == "fork":
            # the best sequences replace others
            p = randperm(N)
            s["dst"] = p[:c["pairs"]].to(torch.int32)
            rest = p[c["pairs"]:]
            s["src"] = rest[torch.arange(c["pairs"], device="cuda") % rest.numel()].to(torch.int32)
    return s


# ---------------------------------------------------------------- mm3fa's calls

def _own(s):
    c = s["case"]
    cache = s.get("cache")
    if cache is None:
        import os
        import sys
        at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "minimaxmusic.cpp_b200")
        if at not in sys.path:
            sys.path.insert(0, at)
        import mm3fa
        cache = s["cache"] = mm3fa.Kv8Cache(s["k"], s["v"], s["k_scale"], s["v_scale"])
    if c["op"] == "attend":
        cache.attend(0, s["q"], s["table"], s["kv_len"], c["D"] ** -0.5, out=s["out"], q_len=s["q_len"], causal=True)
        return s["out"]
    if c["op"] == "append":
        cache.append(0, s["k_new"], s["v_new"], s["table"], s["kv_len"])
        cache.read(0, s["k_out"], s["v_out"], s["table"], s["first"], s["rows"])
        return {"k": s["k_out"], "v": s["v_out"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    if c["op"] == "fork":
        cache.fork(s["src"], s["dst"], s["table"], s["kv_len"], s["refs"], s["table_out"], s["kv_len_out"], s["refs_out"],
                   deep=c["deep"])
    else:
        cache.compact(s["table"], s["refs"], s["table_out"], s["refs_out"])
        s["kv_len_out"].copy_(s["kv_len"])
    return _pool_state(s)


def _pool_state(s):
    return {k: s[k] for k in ("table_out", "kv_len_out", "refs_out", "k", "v", "k_scale", "v_scale")}


# ---------------------------------------------------------------- the plain form

def _values(pool, scale, table):
    """F32 values [N, Hkv, max_pages * P, D] of the pages that a table names."""
    t = table.clamp(min=0).long()
    x = pool[t].float() * scale[t][..., None, None]
    N, n, Hkv, P, D = x.shape
    return x.transpose(1, 2).reshape(N, Hkv, n * P, D)


def _plain_attend(s):
    c, q = s["case"], s["q"]
    N, H, n_q, D = q.shape
    Hkv = c["Hkv"]
    k, v = (_values(s[x][0], s[x + "_scale"][0], s["table"]) for x in ("k", "v"))
    n_kv = k.shape[2]
    sc = (q.float().reshape(N, Hkv, H // Hkv * n_q, D) @ k.transpose(2, 3)) * D ** -0.5
    q_len = s["q_len"] if s["q_len"] is not None else torch.full_like(s["kv_len"], n_q)
    row = torch.arange(n_q, device=q.device)
    seen = s["kv_len"][:, None] - q_len[:, None] + row + 1  # [N, n_q]
    hidden = torch.arange(n_kv, device=q.device) >= seen[..., None]  # [N, n_q, n_kv]
    sc = sc.view(N, H, n_q, n_kv).masked_fill_(hidden[:, None], float("-inf"))
    m = sc.amax(-1, keepdim=True).clamp(min=-3e38)
    e = sc.sub_(m).exp_()
    l = e.sum(-1, keepdim=True)
    o = (e.view(N, Hkv, -1, n_kv) @ v).view(N, H, n_q, D) / torch.where(l > 0, l, 1)
    live = (row < q_len[:, None])[:, :, None, None]
    return torch.where(live, o.transpose(1, 2).to(s["out"].dtype), s["out"])


def _plain_append_one(pool, scale, x, table, start):
    """Writes x [N, Hkv, T, D] behind the first start[s] tokens of each sequence's pages."""
    N, Hkv, T, D = x.shape
    P, dev = pool.shape[2], x.device
    first = torch.div(start, P, rounding_mode="floor").long()
    j = torch.arange(_pages(T, P) + 1, device=dev)
    slot = (first[:, None] + j).clamp(max=table.shape[1] - 1)
    page = table.gather(1, slot).clamp(min=0).long()  # [N, J]
    pos = (first[:, None] + j)[..., None] * P + torch.arange(P, device=dev)  # [N, J, P]
    idx = pos - start[:, None, None]
    new = ((idx >= 0) & (idx < T))[:, :, None, :, None]
    held = (idx < 0)[:, :, None, :, None]
    xn = x.float().transpose(1, 2)  # [N, T, Hkv, D]
    rows = xn.gather(1, idx.clamp(0, T - 1).reshape(N, -1, 1, 1).expand(-1, -1, Hkv, D)).view(N, -1, P, Hkv, D).transpose(2, 3)
    amax = torch.where(new, rows.abs(), 0).amax((3, 4))  # [N, J, Hkv]
    before = torch.where(held.any(3).squeeze(-1), scale[page], 0)
    d = torch.maximum(before, amax / torch.tensor(127.0, device=dev))
    # borders between two codes decide in 64 bits: the quotients there are exact enough
    d64 = torch.where(d > 0, d, 1).double()[..., None, None]
    code = pool[page]
    kept = (code.double() * before.double()[..., None, None] / d64).round()
    fresh = (rows.double() / d64).round().clamp(-127, 127)
    code = torch.where(new, fresh, torch.where(held, kept, code.double())).to(torch.int8)
    touched = new.any(3).view(N, -1)
    pool[page[touched]] = code[touched]
    scale[page[touched]] = d[touched]


def _plain_read(pool, scale, table, start, n, out):
    x = _values(pool, scale, table)
    row = torch.arange(out.shape[2], device=x.device)
    pos = (start[:, None].long() + row).clamp(max=x.shape[2] - 1)
    x = x.gather(2, pos[:, None, :, None].expand(-1, x.shape[1], -1, x.shape[3]))
    return torch.where((row < n[:, None])[:, None, :, None], x, out)


def _plain_append(s):
    for x in ("k", "v"):
        _plain_append_one(s[x][0], s[x + "_scale"][0], s[x + "_new"], s["table"], s["kv_len"])
    k, v = (_plain_read(s[x][0], s[x + "_scale"][0], s["table"], s["first"], s["rows"], s[x + "_out"]) for x in ("k", "v"))
    return {"k": k, "v": v, "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def _move(s, src, dst):
    for x in ("k", "v", "k_scale", "v_scale"):
        s[x][:, dst] = s[x][:, src]


def _plain_fork(s):
    P, table, length, refs = s["case"]["P"], s["table"], s["kv_len"], s["refs"]
    src, dst = s["src"].long(), s["dst"].long()
    j = torch.arange(table.shape[1], device=table.device)
    rows, old = table[src], table[dst]
    n = length[src].long()
    has = j * P < n[:, None]
    fresh = has if s["case"]["deep"] else has & ((j + 1) * P > n[:, None])
    # fresh pages go to the sequences in their order, lowest page first
    rank = torch.argsort(dst)
    need = torch.zeros(table.shape, dtype=torch.bool, device=table.device)
    need[dst] = fresh
    at = need.nonzero()
    free = (refs == 0).nonzero().view(-1)[:at.shape[0]]
    out = table.clone()
    out[dst] = torch.where(has, rows, -1)
    came_from = out[at[:, 0], at[:, 1]].long()
    out[at[:, 0], at[:, 1]] = free.to(torch.int32)
    count = refs.clone()
    count.index_add_(0, old[old >= 0].long(), torch.full_like(old[old >= 0], -1))
    named = out[dst[rank]]
    count.index_add_(0, named[named >= 0].long(), torch.ones_like(named[named >= 0]))
    _move(s, came_from, free)
    s["table_out"].copy_(out)
    s["refs_out"].copy_(count)
    s["kv_len_out"].copy_(length)
    s["kv_len_out"][dst] = length[src]
    return _pool_state(s)


def _plain_compact(s):
    refs, table = s["refs"], s["table"]
    live = refs > 0
    n_live = int(live.sum())
    i = torch.arange(refs.numel(), device=refs.device)
    holes, movers = (~live & (i < n_live)).nonzero().view(-1), (live & (i >= n_live)).nonzero().view(-1)
    to = i.clone()
    to[movers] = holes
    _move(s, movers, holes)
    count = refs.clone()
    count[holes] = refs[movers]
    count[n_live:] = 0
    s["table_out"].copy_(torch.where(table >= 0, to[table.clamp(min=0).long()].to(torch.int32), -1))
    s["refs_out"].copy_(count)
    s["kv_len_out"].copy_(s["kv_len"])
    return _pool_state(s)


_PLAIN = {"attend": _plain_attend, "append": _plain_append, "fork": _plain_fork, "compact": _plain_compact}


def run(state):
    if own:
        return _own(state)
    return _PLAIN[state["case"]["op"]](state)


# ---------------------------------------------------------------- what it takes, and what is right

def work(case):
    c = case
    N, Hkv, D, P = c["N"], c["Hkv"], c["D"], c["P"]
    esz = 4 if c.get("dtype") == "f32" else 2
    if c["op"] == "attend":
        held = _lengths(c["kv_min"], c["kv_max"], N)
        q_len = [min(n, h) for n, h in zip(_lengths(1, c["n_q"], N), held)] if c["ragged_q"] else [c["n_q"]] * N
        pairs = sum(q * (h - q) + q * (q + 1) // 2 for q, h in zip(q_len, held))
        nbytes = sum(2 * Hkv * (h * D + 4 * _pages(h, P)) + 4 * _pages(h, P) for h in held)
        return {"bytes": nbytes + 2 * sum(q_len) * c["H"] * D * esz, "flops": 4 * D * c["H"] * pairs}
    if c["op"] == "append":
        # new rows read once, their codes written, read back and returned as F32 with the codes of the page's other rows
        new = 2 * N * c["T"] * Hkv * D
        before = 2 * sum(h % P for h in _lengths(c["start_min"], c["start_max"], N)) * Hkv * D
        return {"bytes": new * (esz + 1 + 1 + 4) + before * (1 + 4), "flops": 4 * new}
    L, held = c["L"], _lengths(c["kv_min"], c["kv_max"], N)
    page = 2 * L * Hkv * (P * D + 4)
    if c["op"] == "fork":
        # the pages of an average sequence, or one page, for each pair: read and written
        moved = c["pairs"] * (sum(_pages(h, P) for h in held) / N if c["deep"] else 1)
    else:
        used = sum(_pages(h, P) for h in held)
        moved = used * c["holes"]
    return {"bytes": 2 * moved * page + 16 * N * _pages(max(held), P), "flops": 0}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attend":
        return _exact_attend(s)
    if case["op"] == "append":
        return _exact_append(s)
    return None  # copies and counts: compared for equality


def _exact_attend(s):
    c = s["case"]
    P, D, group = c["P"], c["D"], c["H"] // c["Hkv"]
    out = s["out"].double()
    lens = s["kv_len"].tolist()
    q_lens = s["q_len"].tolist() if s["q_len"] is not None else [c["n_q"]] * c["N"]
    for i, (n, m) in enumerate(zip(lens, q_lens)):
        pages = s["table"][i, :_pages(n, P)].long()
        for h in range(c["Hkv"]):
            k, v = ((s[x][0, pages, h].double() * s[x + "_scale"][0, pages, h].double()[:, None, None]).view(-1, D)[:n] for x in ("k", "v"))
            for r in range(0, m, 256):
                rows = torch.arange(r, min(m, r + 256), device=k.device)
                q = s["q"][i, h * group:(h + 1) * group, r:r + rows.numel()].double()
                a = torch.einsum("hrd,kd->hrk", q, k) / D ** 0.5
                a += torch.where(torch.arange(n, device=k.device) <= (n - m + rows)[:, None], 0.0, float("-inf"))
                seen = (n - m + rows) >= 0
                w = torch.softmax(torch.where(seen[None, :, None], a, 0.0), -1) * seen[None, :, None]
                out[i, r:r + rows.numel(), h * group:(h + 1) * group] = torch.einsum("hrk,kd->rhd", w, v)
    return out


def _exact_append(s):
    c = s["case"]
    P, T = c["P"], c["T"]
    got = {}
    for x in ("k", "v"):
        res = torch.zeros(c["N"], c["Hkv"], T + P - 1, c["D"], dtype=torch.float64, device="cuda")
        scales = s[x + "_scale"].double()
        for i, at in enumerate(s["kv_len"].tolist()):
            for j in range(at // P, (at + T - 1) // P + 1):
                page = int(s["table"][i, j])
                a, b = max(at, j * P) - at, min(at + T, j * P + P) - at
                rows = s[x + "_new"][i, :, a:b].double()
                d = (rows.abs().amax((1, 2)) / 127).float().double()  # the scale is held in F32
                held = max(0, at - j * P)  # only in the first page
                if held:
                    before = scales[0, page].clone()
                    d = torch.maximum(d, before)
                    old = s[x][0, page, :, :held].double() * before[:, None, None]
                    res[i, :, :held] = (old / d[:, None, None]).round() * d[:, None, None]
                scales[0, page] = d
                d, a, b = d[:, None, None], a + at % P, b + at % P
                res[i, :, a:b] = torch.where(d > 0, (rows / d).round().clamp(-127, 127) * d, 0.0)
        got[x], got[x + "_scale"] = res, scales
    return {"k": got["k"], "v": got["v"], "k_scale": got["k_scale"], "v_scale": got["v_scale"]}
