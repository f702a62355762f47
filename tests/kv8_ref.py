"""Plain references of the 8-bit paged cache's operators (numpy and torch in 64 bits) and test inputs."""
from __future__ import annotations

import numpy as np
import torch


class State:
    """A cache of L layers with scattered pages: sequence s holds lens[s] tokens and has pages for room[s]."""

    def __init__(self, lens, Hkv, D, P, L=1, room=None, spare=5, seed=0, device="cpu"):
        g = torch.Generator().manual_seed(seed)
        room = room or lens
        used = [-(-n // P) for n in room]
        self.N, self.P, self.Hkv, self.D, self.L = len(lens), P, Hkv, D, L
        self.n_pages = sum(used) + spare
        shape = (L, self.n_pages, Hkv, P, D)
        self.k = (torch.randn(shape, generator=g) * 32).round().clamp(-127, 127).to(torch.int8)
        self.v = (torch.randn(shape, generator=g) * 32).round().clamp(-127, 127).to(torch.int8)
        self.ks = 0.03 * torch.exp(0.3 * torch.randn(shape[:3], generator=g))
        self.vs = 0.016 * torch.exp(0.7 * torch.randn(shape[:3], generator=g))
        order = torch.randperm(self.n_pages, generator=g)[:sum(used)].to(torch.int32)
        self.table = torch.full((self.N, max(used + [1])), -1, dtype=torch.int32)
        at = 0
        for i, n in enumerate(used):
            self.table[i, :n] = order[at:at + n]
            at += n
        self.refs = torch.zeros(self.n_pages, dtype=torch.int32)
        self.refs[order.long()] = 1
        self.len = torch.tensor(lens, dtype=torch.int32)
        self.g = g
        for x in ("k", "v", "ks", "vs", "table", "refs", "len"):
            setattr(self, x, getattr(self, x).to(device))

    def cache(self):
        import mm3fa

        return mm3fa.Kv8Cache(self.k, self.v, self.ks, self.vs)

    def randn(self, *shape):
        return torch.randn(*shape, generator=self.g).to(self.k.device)


def keys_of(pool, scale, table_row, n, n_pages):
    """float64 values [Hkv, n, D] of a sequence's first n tokens, and which of them are there."""
    P = pool.shape[2]
    pages = [int(x) for x in table_row[:-(-n // P)].tolist()]
    ok = [0 <= p < n_pages for p in pages]
    at = torch.tensor([p if o else 0 for p, o in zip(pages, ok)], dtype=torch.long, device=pool.device)
    x = pool[at].double() * scale[at].double()[..., None, None]  # [J, Hkv, P, D]
    x = x.transpose(0, 1).reshape(pool.shape[1], len(pages) * P, pool.shape[3])[:, :n]
    there = torch.tensor(ok, dtype=torch.bool, device=pool.device).repeat_interleave(P)[:n]
    return x, there


def attend(st, layer, q, scale, q_len=None, causal=True, softcap=0.0, out=None, kv_len=None):
    """float64 result (N, n_q, H, D) and a bound for each row's F32 arithmetic, per value."""
    N, H, n_q, D = q.shape
    G = H // st.Hkv
    res = torch.zeros(N, n_q, H, D, dtype=torch.float64, device=q.device) if out is None else out.double().clone()
    f32 = torch.zeros(N, n_q, H, 1, dtype=torch.float64, device=q.device)
    p16 = torch.zeros(N, n_q, H, 1, dtype=torch.float64, device=q.device)
    lens = (st.len if kv_len is None else kv_len).tolist()
    for s in range(N):
        n = max(0, min(lens[s], st.table.shape[1] * st.P))
        m = n_q if q_len is None else max(0, min(int(q_len[s]), n_q))
        if m == 0:
            continue
        k, there = keys_of(st.k[layer], st.ks[layer], st.table[s], n, st.n_pages)
        v, _ = keys_of(st.v[layer], st.vs[layer], st.table[s], n, st.n_pages)
        qs = q[s, :, :m].double().reshape(st.Hkv, G, m, D)
        sc = torch.einsum("hgrd,hkd->hgrk", qs, k) * scale
        # q and k products: 22 bits of q, D additions in F32 (2^-24 each of the sum of magnitudes), the scalings
        mag = torch.einsum("hgrd,hkd->hgrk", qs.abs(), k.abs()) * abs(scale)
        if softcap:
            sc = softcap * torch.tanh(sc / softcap)
        row = torch.arange(m, device=q.device)
        seen = there[None, :].expand(m, n).clone()
        if causal:
            seen &= torch.arange(n, device=q.device)[None] < (n - (m - 1 - row))[:, None]
        sc = sc.masked_fill(~seen, float("-inf"))
        any_ = seen.any(-1)
        w = torch.softmax(torch.where(any_[:, None], sc, 0.0), -1) * any_[:, None] if n else sc.new_zeros(sc.shape)
        o = torch.einsum("hgrk,hkd->hgrd", w, v)
        res[s, :m] = o.permute(2, 0, 1, 3).reshape(m, H, D)
        if n == 0:
            continue
        vmax = torch.einsum("hgrk,hk->hgr", w, v.abs().amax(-1))
        big = mag.masked_fill(~seen, 0).amax(-1)
        # a score off by e changes each weight by e and their sum by e at most; tanh and 2^x: 4 ulp; the score's own
        # rounding in the exponent; sums of n weights and products
        e = big * (D + 16) * 2.0 ** -24 + (big + 8 + n) * 2.0 ** -22
        f32[s, :m] = (2 * e * v.abs().amax((-1, -2))[:, None, None]).permute(2, 0, 1).reshape(m, H, 1)
        p16[s, :m] = (2.0 ** -11 * vmax).permute(2, 0, 1).reshape(m, H, 1)
    return res, f32, p16


def check_attend(got, ref, f32, p16, dtype, what=""):
    """F32 results within F32's arithmetic; 16-bit ones within half a step of the result, half a step (2^-12,
    counted twice: up and down) of each weight, and F32's arithmetic."""
    tol = f32 + 1e-30
    if dtype != torch.float32:
        tol = tol + p16 + ref.abs() * torch.finfo(dtype).eps / 2 * 1.01
        tol = tol + torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    off = (got.double() - ref).abs()
    assert torch.isfinite(got).all(), f"{what}: values that are not finite"
    worst = (off / tol).max().item() if off.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.3f} times the bound"
    return worst


def append_one(codes, scales, x, table_row, start, n, P):
    """In place on numpy codes [n_pages, Hkv, P, D], scales [n_pages, Hkv]; x float32 [Hkv, T, D]."""
    n_pages = codes.shape[0]
    if start < 0 or n <= 0:
        return
    for j in range(start // P, (start + n - 1) // P + 1):
        if j >= len(table_row) or not 0 <= table_row[j] < n_pages:
            continue
        page = table_row[j]
        a, b = max(start, j * P), min(start + n, (j + 1) * P)
        rows = x[:, a - start:b - start]
        for h in range(codes.shape[1]):
            r = rows[h].astype(np.float64)
            fin = np.abs(r[np.isfinite(r)])
            d = np.float32(np.float32(fin.max() if fin.size else 0.0) / np.float32(127.0))
            held = a - j * P
            if held:
                before = scales[page, h]
                d = max(before, d)
                if d > before:
                    c = codes[page, h, :held].astype(np.float64)
                    codes[page, h, :held] = np.rint(c * float(before) / float(d)).astype(np.int8)
            scales[page, h] = d
            with np.errstate(all="ignore"):
                q = np.rint(r / float(d)) if d > 0 else np.where(np.isinf(r), np.sign(r) * 127, 0.0)
                q = np.where(np.isnan(r), 0.0, np.clip(q, -127, 127))
            codes[page, h, a - j * P:b - j * P] = q.astype(np.int8)


def fork(table, length, refs, src, dst, P, deep):
    """(table, length, refs, [(from, to)], failed) as new lists from lists."""
    N, mp, n_pages = len(table), len(table[0]), len(refs)
    win = {}
    for i, d in enumerate(dst):
        s = -1 if src is None else src[i]
        if 0 <= d < N and -1 <= s < N and d not in win:
            win[d] = s
    win = {d: s for d, s in win.items() if s != d}
    free = [p for p in range(n_pages) if refs[p] == 0]
    t2, l2, r2, moves = [list(r) for r in table], list(length), list(refs), []
    for d in sorted(win):
        s = win[d]
        n = 0 if s < 0 else max(0, min(length[s], mp * P))
        row = [-1] * mp
        for j in range(-(-n // P)):
            page = table[s][j]
            if 0 <= page < n_pages:
                if deep or (j + 1) * P > n:
                    if not free:
                        return [list(r) for r in table], list(length), list(refs), [], True
                    to = free.pop(0)
                    moves.append((page, to))
                    r2[to] = 1
                    page = to
                else:
                    r2[page] += 1
            row[j] = page
        for page in table[d]:
            if 0 <= page < n_pages:
                r2[page] -= 1
        t2[d], l2[d] = row, 0 if s < 0 else length[s]
    return t2, l2, r2, moves, False


def compact(table, refs):
    n_pages = len(refs)
    L = sum(r > 0 for r in refs)
    holes = [p for p in range(L) if refs[p] == 0]
    moves = list(zip([p for p in range(L, n_pages) if refs[p] > 0], holes))
    to = dict(moves)
    t2 = [[to.get(p, p) if 0 <= p < n_pages else -1 for p in row] for row in table]
    r2 = [refs[p] if p < L else 0 for p in range(n_pages)]
    for a, b in moves:
        r2[b] = refs[a]
    return t2, r2, moves


def reserve(table, refs, n_tok, P):
    t2, r2 = [list(r) for r in table], list(refs)
    free = [p for p in range(len(refs)) if refs[p] == 0]
    for s, n in enumerate(n_tok):
        need = -(-max(0, n) // P)
        if need > len(table[0]):
            return table, refs, True
        for j in range(need):
            if t2[s][j] < 0:
                if not free:
                    return table, refs, True
                t2[s][j] = free.pop(0)
                r2[t2[s][j]] = 1
    return t2, r2, False
