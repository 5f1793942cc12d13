"""Inputs and float64 results of the paged cache's ops, for their CPU and GPU tests.

Errors are bounded by arithmetic. Attention: P enters the second product rounded to u_p (relative
half a step: bf16 2^-8, fp16 2^-11, nothing in fp32 and over a 4-bit cache but in bf16), the output
is rounded to u, and the fp32 sums of d products (then a score's error, so a probability's relative
one) and of L terms each add 2^-23 a term, an addition of the matrix cores being no worse than one
whole step. So |o - exact| <= u |o| + (u_p + e) sum(p |v|), with
e = 2^-23 (2 (d + 8) max_j scale sum|q k_j| + L + 32).
"""

from __future__ import annotations

import math

import torch

from popcorn_amd.compat import references as R

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def cache_of(pages, kv_heads, page_size, d, dtype, seed, device="cpu"):
    g = torch.Generator().manual_seed(seed)
    return tuple(torch.randn(pages, kv_heads, page_size, d, generator=g).to(dtype).to(device) for _ in range(2))


def mxfp4_of(cache):
    """codes and scales of rows [pages, kv_heads, page_size, d]."""
    codes, scales = R.mxfp4_encode(cache)
    return codes, scales.transpose(-1, -2).contiguous()


def values_of(codes, scales):
    return R.mxfp4_decode(codes, scales.transpose(-1, -2))


def table_of(lens, page_size, pages, width, seed, fill=0):
    """Distinct pages for every sequence, in any order."""
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(pages, generator=g).int()
    table = torch.full((len(lens), width), fill, dtype=torch.int32)
    at = 0
    for i, n in enumerate(lens):
        need = -(-n // page_size)
        table[i, :need] = order[at:at + need]
        at += need
    return table


def exact(q, k_rows, v_rows, table, lens, cu, causal, scale, d_terms=None):
    """float64 (o, what sum(p |v|) is, the largest scale * sum|q k|) per output row; k_rows, v_rows the cache's values."""
    q = q.double()
    pages, kv_heads, ps, d = k_rows.shape
    total, hq, _ = q.shape
    group = hq // kv_heads
    scale = d ** -0.5 if scale is None else scale
    o, mass = torch.zeros_like(q), torch.zeros_like(q)
    size = torch.zeros(total, hq, dtype=torch.float64)
    cuts = list(range(total + 1)) if cu is None else cu.tolist()
    for i, length in enumerate(lens):
        length = min(max(length, 0), table.shape[1] * ps)
        n = cuts[i + 1] - cuts[i]
        key = torch.arange(length)
        page = table[i].long()[key // ps]
        there = (page >= 0) & (page < pages)
        k = k_rows[page.clamp(0, pages - 1), :, key % ps].double()
        v = v_rows[page.clamp(0, pages - 1), :, key % ps].double()
        for t in range(n):
            row = cuts[i] + t
            seen = torch.nonzero(there & (key < (length - n + t + 1 if causal else length)))[:, 0]
            if seen.numel() == 0:
                continue
            for h in range(kv_heads):
                kk, vv = k[seen, h], v[seen, h]
                qq = q[row, h * group:(h + 1) * group]
                p = torch.softmax(qq @ kk.T * scale, dim=-1)
                o[row, h * group:(h + 1) * group] = p @ vv
                mass[row, h * group:(h + 1) * group] = p @ vv.abs()
                size[row, h * group:(h + 1) * group] = (qq.abs() @ kk.abs().T * abs(scale)).amax(-1)
    return o, mass, size


def check(got, want, dtype, d, longest, mxfp4=False, what=""):
    o, mass, size = want
    u = HALF_STEP[dtype]
    u_p = 0.0 if dtype == torch.float32 or (mxfp4 and dtype != torch.bfloat16) else u
    e = 2.0 ** -23 * (2 * (d + 8) * size[..., None] + longest + 32)
    limit = u * o.abs() + (u_p + e) * mass + 2.0 ** -24 * (1 if dtype == torch.float16 else 0)
    off = (got.cpu().double() - o).abs()
    bad = ~(off <= limit)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} values off, worst {float((off / limit.clamp(min=1e-300)).nan_to_num(math.inf).max()):.2f} "
                           f"times the limit, first at {torch.nonzero(bad)[0].tolist()}")
