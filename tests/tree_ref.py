"""References in 64 bits of the operators of decoding with a tree of drafted tokens, and a bound for the attention's error.

A relative error e_j of the weight of key j moves a result row o = sum_j w_j v_j by w_j e_j (v_j - o).  The inputs are
random, so the errors of different keys are independent and their squares add:

    |err| <= e * sqrt(sum_j w_j^2 |v_j|^2) + t * |o|        (2-norms over the head dimension)

With scores |s| <= 5 in natural units (they are normal, around 1), where the result is F32 or q has more bits than the
cache's type holds (two parts of each operand, 22 bits in F16, 16 in BF16):

    F16 cache   q, off by 2^-22 of each element: 5 * 2^-22 in the score; the score's scalings, four F32 roundings in log2
                units: 4 * 5 * 1.45 * 2^-24; its sum, 16 additions truncated at 2^-23 of a partial sum, of 2 on average:
                16 * 2 * 2^-23; 2^x and the pair that holds the weight: 3 * 2^-22.  Together less than e = 2^-17
    BF16 cache  q, off by 2^-17 of each element: 5 * 2^-17, and the weight's pair 2^-17: e = 2^-14
    t           16 truncated additions a tile, for two parts: 2^-18

and else the weights have the cache's type: e = half its step more.  (On CUDA cores all is F32, e and t below these.)
A result in fewer bits is off by half its type's step more.
"""
from __future__ import annotations

import torch

Q8 = "q8_0"


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def q8_values(x):
    """(.., bytes) of Q8_0 blocks -> F64 values."""
    b = x.reshape(*x.shape[:-1], -1, 34)
    d = b[..., :2].contiguous().view(torch.float16).double()
    return (b[..., 2:].contiguous().view(torch.int8).double() * d).reshape(*x.shape[:-1], -1)


def values(x):
    return q8_values(x) if x.dtype is torch.uint8 else x.double()


def ancestors(parents, i):
    """Node i and its ancestors; a parent outside [0, i) is none."""
    found = []
    while True:
        found.append(i)
        p = int(parents[i])
        if not 0 <= p < i:
            return found
        i = p


def attend(q, k, v, parents, n_nodes, kv_len, scale, out, softcap=0.0):
    """(result [N, T, H, D] in 64 bits over `out`'s values, sqrt(sum w^2 |v|^2) [N, T, H])."""
    N, H, T, D = q.shape
    Hkv, rows = k.shape[1], k.shape[2]
    res = out.double().clone()
    spread = torch.zeros(N, T, H, dtype=torch.float64, device=q.device)
    for s in range(N):
        tree = s % parents.shape[0]
        L = min(max(int(kv_len[s]), 0), rows)
        m = T if n_nodes is None else min(max(int(n_nodes[tree]), 0), T)
        for i in range(m):
            keys = list(range(L)) + sorted(L + j for j in ancestors(parents[tree].tolist(), i) if L + j < rows)
            if not keys:
                res[s, i] = 0.0
                continue
            kk, vv = values(k[s][:, keys]), values(v[s][:, keys])
            a = torch.einsum("hgd,hkd->hgk", q[s, :, i].double().view(Hkv, H // Hkv, D), kk) * scale
            if softcap:
                a = softcap * torch.tanh(a / softcap)
            w = torch.softmax(a, -1)
            res[s, i] = torch.einsum("hgk,hkd->hgd", w, vv).reshape(H, D)
            spread[s, i] = torch.einsum("hgk,hk->hg", w * w, (vv * vv).sum(-1)).sqrt().reshape(H)
    return res, spread


def bound(want, spread, q, k, out):
    two = out.dtype is torch.float32 or (q.dtype is not k.dtype)
    e = 2.0 ** -14 if k.dtype is torch.bfloat16 else 2.0 ** -17
    if not two:
        e = e + half_step(k.dtype)
    h = 0.0 if out.dtype is torch.float32 else half_step(out.dtype)
    tiny = torch.finfo(out.dtype).smallest_normal * want.shape[-1] ** 0.5
    return e * spread + (2.0 ** -18 + h) * want.norm(dim=-1) + tiny


def check(got, want, spread, q, k):
    assert torch.isfinite(got).all()
    ratio = ((got.double() - want).norm(dim=-1) / bound(want, spread, q, k, got)).max().item()
    assert ratio <= 1.0, f"{ratio:.3f} times the bound"


def verify(logits, tokens, accept, sample, parents, n_nodes, draft, temperature):
    """The walk, tree by tree, in 64 bits: lists of (path, token)."""
    got = []
    n, T, V = logits.shape
    x = logits.double().cpu()
    x = torch.where(x.isnan(), float("-inf"), x).clamp(max=torch.finfo(torch.float32).max)
    d = None if draft is None else torch.nan_to_num(draft.double().cpu(), nan=0.0, posinf=float("inf")).clamp(min=0)
    for t in range(n):
        m = T if n_nodes is None else min(max(int(n_nodes[t]), 0), T)
        if m == 0:
            got.append(([], -1))
            continue
        par, tok = parents[t].tolist(), tokens[t].tolist()
        cur, path = 0, [0]
        while True:
            row = x[t, cur]
            dead = not (row > float("-inf")).any()
            kids = [i for i in range(cur + 1, m) if par[i] == cur and 0 <= tok[i] < V]
            nxt = None
            if temperature == 0 or dead:
                best = int(row.argmax()) if not dead else -1
                best = int((row == row.max()).nonzero()[0]) if not dead else -1
                nxt = next((i for i in kids if tok[i] == best), None)
                left = None
            else:
                p = torch.softmax(row / temperature, -1)
                left, mass = p.clone(), 1.0
                for i in kids:
                    q = torch.zeros(V, dtype=torch.float64) if d is None else d[t, cur]
                    if d is None:
                        q[tok[i]] = 1.0
                    if float(accept[t, i]) * float(q[tok[i]]) * mass < float(left[tok[i]]):
                        nxt = i
                        break
                    left = (left - mass * q).clamp(min=0)
                    mass = float(left.sum())
            if nxt is None:
                break
            cur = nxt
            path.append(cur)
        if left is None:
            got.append((path, best))
            continue
        left = left if mass > 0 else p
        at = left.cumsum(-1)
        u = min(max(float(sample[t]), 0.0), 1 - 2.0 ** -24) if float(sample[t]) == float(sample[t]) else 0.0
        got.append((path, int((at > u * at[-1]).nonzero()[0])))
    return got


def commit(slabs, path, n_path, kv_len):
    """Copies of the slabs (layers of (N, Hkv, rows, D)) with the rows moved, and the new lengths."""
    out, lens = [], kv_len.clone()
    T = path.shape[1]
    for s in range(kv_len.shape[0]):
        t, L, n, last = s % path.shape[0], int(kv_len[s]), 0, -1
        rows = slabs[0].shape[2]
        for at in path[t, :max(0, min(int(n_path[t]), T))].tolist():
            if L < 0 or at <= last or at >= T or L + at >= rows:
                break
            last, n = at, n + 1
        lens[s] = L + n
    for x in slabs:
        y = x.clone()
        for s in range(kv_len.shape[0]):
            L, n = int(kv_len[s]), int(lens[s] - kv_len[s])
            if n:
                y[s][:, L:L + n] = x[s][:, (L + path[s % path.shape[0], :n].long())]
        out.append(y)
    return out, lens
