"""Attention over a paged cache from its definition (include/kvattn.h) in 64
bits, one sequence, node and head at a time, with the bounds that rounding
sets for a result computed in fewer bits."""
from __future__ import annotations

import math

import torch


def visible(parents: list[int] | None, nodes: int) -> list[set[int] | None]:
    """the nodes that each node sees; None for a padding node"""
    ok = [parents is None or -1 <= parents[j] < j for j in range(nodes)]
    out: list[set[int] | None] = []
    for j in range(nodes):
        if not ok[j]:
            out.append(None)
            continue
        up = j - 1 if parents is None else parents[j]
        out.append({j} | (out[up] if up >= 0 and ok[up] else set()))
    return out


def attention(q, k_pages, v_pages, table, lens, q_offsets, parents=None, rows=None, scale=None, k_scale=1.0, v_scale=1.0):
    """k_pages, v_pages: [pages, block, kv heads, dim] float64.  Returns out,
    lse, and per element the bounds out_tol, lse_tol of a kernel that rounds
    the weights and the result to q's type and holds all else in 32 bits:

    u = eps / 2 of q's type.  A score is a sum of dim products in 32 bits, off
    by (dim + 2) 2^-24 sum |q k|, and the exponential's argument and value add
    2^-23 |s| + 2^-21: d in all, relative to a weight.  Each weight is rounded
    (u), the two sums over n positions lose n 2^-24 each, the result is
    rounded (u |out|).  With A the weighted mean of |v|:
    out_tol = u |out| + t + (u + 2 d + 2 n 2^-24) A,  lse_tol = 2 d + n 2^-24 + 2^-22 |lse|,
    where t = u times the smallest normal number of q's type: below it the
    type's steps no longer shrink with the value (fp16: 2^-24, half a step 2^-25).
    """
    u = torch.finfo(q.dtype).eps / 2
    total, heads, dim = q.shape
    group = heads // k_pages.shape[2]
    scale = dim ** -0.5 if scale is None else scale
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.full((total, heads), -math.inf, dtype=torch.float64, device=q.device)
    out_tol, lse_tol = torch.zeros_like(out), torch.zeros_like(lse)
    block = k_pages.shape[1]
    for b in range(len(q_offsets) - 1):
        first, nodes = q_offsets[b], q_offsets[b + 1] - q_offsets[b]
        r = b if rows is None else rows[b]
        n = lens[r]
        before = n - nodes
        if nodes == 0:
            continue
        ids = torch.tensor(table[r][:-(-n // block)], device=q.device, dtype=torch.long)
        k = k_pages[ids].flatten(0, 1)[:n] * k_scale
        v = v_pages[ids].flatten(0, 1)[:n] * v_scale
        sees = visible(parents[first:first + nodes] if parents is not None else None, nodes)
        for j in range(nodes):
            if sees[j] is None:
                continue
            at = torch.tensor(list(range(before)) + sorted(before + x for x in sees[j]), device=q.device)
            for h in range(k.shape[1]):
                x = q[first + j, h * group:(h + 1) * group].double()
                kk, vv = k[at, h], v[at, h]
                s = scale * x @ kk.T
                m = s.amax(-1, keepdim=True)
                w = (s - m).exp()
                z = w.sum(-1, keepdim=True)
                o = (w / z) @ vv
                d = (scale * (x.abs() @ kk.abs().T)).amax(-1, keepdim=True) * (dim + 2) * 2.0 ** -24 \
                    + s.abs().amax(-1, keepdim=True) * 2.0 ** -23 + 2.0 ** -21
                a = (w / z) @ vv.abs()
                sl = slice(h * group, (h + 1) * group)
                out[first + j, sl], lse[first + j, sl] = o, (m + z.log())[:, 0]
                out_tol[first + j, sl] = u * o.abs() + u * torch.finfo(q.dtype).smallest_normal + (u + 2 * d + 2 * len(at) * 2.0 ** -24) * a
                lse_tol[first + j, sl] = 2 * d[:, 0] + len(at) * 2.0 ** -24 + 2.0 ** -22 * lse[first + j, sl].abs()
    return out, lse, out_tol, lse_tol
