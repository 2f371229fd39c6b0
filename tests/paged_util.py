"""Plain implementations of the paged calls in 64 bits (attention, read) and whole numbers (plan), and inputs for their tests."""
from __future__ import annotations

import math

import numpy as np
import torch

CENT = {4: [0.01135, 0.03432, 0.05806, 0.08330, 0.11099, 0.14304, 0.18293, 0.24155], 2: [0.04003, 0.13351]}


def plan(table, stack, count, context, new, finished, page, T):
    """One step by the rules of tq_page_plan, request by request, on Python numbers.  Changes table and stack; returns
    (lens, start, slots, positions, count)."""
    G, width = table.shape
    held = [~c if c < 0 else c for c in context]
    pages = lambda n: -(-n // page)  # noqa: E731
    count = min(max(count, 0), len(stack))
    for g in range(G):
        if finished is not None and finished[g]:
            for j in range(min(pages(held[g]), width)):
                if count < len(stack):
                    stack[count] = table[g, j]
                    count += 1
            held[g] = 0
    lens, start, slots, positions = [], [0], [-1] * T, [-1] * T
    wanted = tokens = taken = 0
    for g in range(G):
        n = max(int(new[g]), 0)
        fits = held[g] + n <= width * page
        need = pages(held[g] + n) - pages(held[g]) if fits else 0
        ok = fits and (n == 0 or (tokens + n <= T and (need == 0 or wanted + need <= count)))
        if ok:
            for j in range(need):
                table[g, pages(held[g]) + j] = stack[count - 1 - wanted - j]
            taken += need
            for i in range(n):
                pos = held[g] + i
                slots[tokens + i] = int(table[g, pos // page]) * page + pos % page
                positions[tokens + i] = pos
        lens.append(held[g] + n if ok else ~held[g])
        wanted += need
        tokens += n
        start.append(min(tokens, T))
    return lens, start, slots, positions, count - taken


def rotation(seed=0):
    gen = torch.Generator().manual_seed(seed)
    q, _ = torch.linalg.qr(torch.randn(128, 128, generator=gen, dtype=torch.float64))
    return q.to(torch.float16).contiguous()


def random_cache(rng, rows, Hkv, bits):
    """Any bytes are codes; norms near those of normal vectors."""
    codes = torch.from_numpy(rng.integers(0, 256, (rows, Hkv * 16 * bits), dtype=np.uint8))
    norms = torch.from_numpy((11.3 * (1 + 0.1 * rng.standard_normal((rows, Hkv)))).astype(np.float16))
    return codes.cuda(), norms.cuda()


def vectors(codes, norms, R, bits):
    """What rows of a cache stand for: [rows, Hkv, 128] in 64 bits."""
    c = torch.tensor([-x for x in reversed(CENT[bits])] + CENT[bits], dtype=torch.float64, device=codes.device)
    n, Hkv = norms.shape
    code = torch.stack([(codes >> s) & ((1 << bits) - 1) for s in range(0, 8, bits)], -1).reshape(n, Hkv, 128)
    return (c[code.long()] * norms.double()[..., None]) @ R.double()


def tables(rng, lens, page, extra_pages=3, extra_columns=1):
    """Pages of a pool dealt out in no order; unused entries name no page at all.  (table, pages in the pool)"""
    need = [-(-max(int(n), 0) // page) for n in lens]
    pool = sum(need) + extra_pages
    order = rng.permutation(pool)
    table = np.full((len(lens), max(need) + extra_columns), -7, np.int32)
    at = 0
    for g, n in enumerate(need):
        table[g, :n] = order[at:at + n]
        at += n
    return torch.from_numpy(table).cuda(), pool


def rows_of(table_row, n, page):
    t = torch.arange(n, device=table_row.device)
    return table_row.long()[t // page] * page + t % page


EPS = 2.0**-11  # half a step of fp16, relative


def attention(q, ck, cv, kn, vn, R, table, lens, start, page, H, Hkv, bits):
    """Causal attention of a ragged batch in 64 bits: queries start[g] .. start[g + 1] - 1 are the last tokens of request g.
    Returns (out [T, H * 128], how far off fp16 arithmetic may be per query and head, in 2-norm [T, H]).

    The kernels round four things to fp16 on the way and the result at the end, each by a relative error of at most EPS, taken as
    independent with a variance of at most EPS^2 / 3: the rotated query's coordinates and K's centroids, which move a score
    s = sum_k q_k c_k n / sqrt(128) by a variance of 2 EPS^2 / 3 sum_k (q_k c_k n)^2 / 128, and with it, s being the logarithm of a
    weight, the weight relatively by as much; the weight (times its norm) by EPS^2 / 3; V's centroids by EPS^2 / 3.  The output moves by the
    sum over the tokens of w_t v_t times those: its squared 2-norm is sum_t w_t^2 |v_t|^2 (their variances' sum) in the mean.  Allowed are six
    times its root, and for the result's rounding, and V's centroids' errors, which are the same wherever a code is, 2 EPS |out|.
    (The prefill kernel for many rows takes the centroids times norms as K's and V's operands, one rounding each as well, and rounds its result before
    the last product, by R: its roundings are 2^-11 / sqrt(3) of it in the mean there and as much at the end, and V's centroids, scaled, are off by 0.22
    of EPS at most: 1.4 EPS |out| together.)
    (fp32 sums of 128 and of n terms, 2^-24 each, and weights below fp16's normal range, 2^-25 each next to a sum of at least 1, are far
    below that: n 2^-25 |v| is added for them.)"""
    T = q.shape[0]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    tol = torch.zeros(T, H, dtype=torch.float64, device=q.device)
    c = torch.tensor([-x for x in reversed(CENT[bits])] + CENT[bits], dtype=torch.float64, device=q.device)
    Rd = R.double()

    def rotated(codes, norms):
        code = torch.stack([(codes >> s) & ((1 << bits) - 1) for s in range(0, 8, bits)], -1).reshape(norms.shape[0], Hkv, 128)
        return c[code.long()] * norms.double()[..., None]

    for g, n in enumerate(lens):
        a, b = start[g], start[g + 1]
        if n <= 0 or a == b:
            continue
        rows = rows_of(table[g], n, page)
        k, v = rotated(ck[rows], kn[rows]), rotated(cv[rows], vn[rows])
        qr = q[a:b].double().view(b - a, Hkv, H // Hkv, 128) @ Rd.T / math.sqrt(128)
        x = torch.einsum("qhgd,khd->hgqk", qr, k)
        pos = n - (b - a) + torch.arange(b - a, device=q.device)
        x = x.masked_fill(torch.arange(n, device=q.device)[None] > pos[:, None], -math.inf)
        w = torch.softmax(x, -1).nan_to_num(0.0)
        out[a:b] = (torch.einsum("hgqk,khd->qhgd", w, v) @ Rd).reshape(b - a, -1)
        spread = (2 / 3 * torch.einsum("qhgd,khd->hgqk", qr.square(), k.square()) + 2 / 3) * EPS**2
        v2 = v.square().sum(-1).T  # [Hkv, n]
        off = 6 * torch.einsum("hgqk,hk->qhg", w.square() * spread, v2).sqrt() + n * 2.0**-25 * v2.amax(1)[None, :, None].sqrt()
        tol[a:b] = off.reshape(b - a, H)
    return out, tol + 2 * EPS * out.view(T, H, 128).norm(dim=-1)


def assert_attention(got, want, what=""):
    out, tol = want
    assert torch.isfinite(got).all(), f"{what}: not finite"
    off = (got.double() - out).view(*tol.shape, 128).norm(dim=-1)
    bad = off > tol
    assert not bad.any(), f"{what}: off by {(off / tol.clamp(min=1e-30)).max().item():.2f} times what roundings explain, at {bad.nonzero()[:4].tolist()}"
