"""A bound for F32 results of the attention over the 8-bit cache that does not grow with the number of keys, and what a
computation with fewer bits would give.

A result row is o = sum_j w_j v_j.  A relative error e_j of the weight of key j moves it by w_j e_j (v_j - o).  The test
inputs are random, so the errors of different keys are independent and their squares add:

    |err| <= e * sqrt(sum_j w_j^2 |v_j|^2) + t * |o|        (2-norms over the head dimension)

with e what one weight's relative error can be and t what all of a row have in common (the sum, and the truncation of what
the tensor core adds to an accumulator, always towards zero).  With scores |s| <= 5 (they are normal, around 1):

    q, off by 2^-22 of each element                          5 * 2^-22   in the score
    the score's scalings, four F32 roundings, in log2 units  4 * 5 * 1.45 * 2^-24
    its sum on the tensor core: 2 * D / 16 <= 16 truncated
    additions of 2^-23 of a partial sum, of 2 on average     16 * 2 * 2^-23 (D = 128)
    2^x, its products and the pair that holds the weight     (1 + 3/4 + 1) * 2^-22
                                                             together less than 32 * 2^-22 = 2^-17, so e = 2^-18 in the mean
    O: 16 truncated additions before a sum in F32            t = 16 * 2^-23 = 2^-19

and where one element of q is far above the others, what the fixed-point form of few rows leaves: no element is off by more
than 2^-30 of the row's largest, which moves a score by 2^-30 max|q| |k_j| scale.
"""
from __future__ import annotations

import torch

import kv8_ref as R


def rows(st, q, s, causal=True):
    """Of sequence s, in 64 bits: scores [Hkv, G, m, n] (-inf: not seen), keys and values [Hkv, n, D]."""
    _, H, m, D = q.shape
    n = int(st.len[s])
    k, there = R.keys_of(st.k[0], st.ks[0], st.table[s], n, st.n_pages)
    v, _ = R.keys_of(st.v[0], st.vs[0], st.table[s], n, st.n_pages)
    sc = torch.einsum("hgrd,hkd->hgrk", q[s].double().reshape(st.Hkv, H // st.Hkv, m, D), k) * D ** -0.5
    seen = there[None, :].expand(m, n)
    if causal:
        seen = seen & (torch.arange(n, device=q.device)[None] < (n - (m - 1 - torch.arange(m, device=q.device)))[:, None])
    return sc.masked_fill(~seen, float("-inf")), k, v


def worst(st, q, got, causal=True):
    """The largest ratio of a row's error to its bound; got [N, m, H, D]."""
    top = 0.0
    for s in range(st.N):
        sc, k, v = rows(st, q, s, causal)
        live = (sc > float("-inf")).any(-1)
        w = torch.softmax(torch.where(live[..., None], sc, 0.0), -1) * live[..., None]
        o = torch.einsum("hgrk,hkd->hgrd", w, v)
        m, D = o.shape[2], o.shape[3]
        err = (got[s].double().permute(1, 0, 2).reshape(o.shape) - o).norm(dim=-1)
        spread = torch.einsum("hgrk,hk->hgr", w * w, (v * v).sum(-1)).sqrt()
        large = q[s].double().abs().amax(-1).reshape(o.shape[:3]) * k.norm(dim=-1).amax(-1)[:, None, None] * D ** -0.5
        bound = (2.0 ** -18 + 2.0 ** -30 * large) * spread + 2.0 ** -19 * o.norm(dim=-1) + 1e-30
        top = max(top, (err / bound).max().item())
    return top


def check(st, q, got, what=""):
    assert torch.isfinite(got).all(), what
    ratio = worst(st, q, got)
    assert ratio <= 1.0, f"{what}: {ratio:.3f} times the bound"
    return ratio


def simulate(st, q, q_type=None, w_type=None):
    """The result, in 64 bits but for q or the weights (over their row's maximum) rounded to a type."""
    N, H, m, D = q.shape
    out = torch.zeros(N, m, H, D, dtype=torch.float64)
    if q_type:
        q = q.to(q_type).double()
    for s in range(N):
        sc, _, v = rows(st, q, s)
        live = (sc > float("-inf")).any(-1, keepdim=True)
        sc = torch.where(live, sc, 0.0)
        p = torch.exp(sc - sc.amax(-1, keepdim=True)) * live
        total = p.sum(-1, keepdim=True)
        if w_type:
            p = p.to(w_type).double()
        o = torch.einsum("hgrk,hkd->hgrd", p / torch.where(total > 0, total, 1.0), v)
        out[s] = o.permute(2, 0, 1, 3).reshape(m, H, D)
    return out
