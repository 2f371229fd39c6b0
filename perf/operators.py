"""The operators of a paged packed KV cache: what they compute, at sizes that serving meets.

The cache is the library's packed one (per token and KV head: 128 codes of 4 or 2 bits in rotated space and an fp16 norm), cut into
pages of `page` consecutive rows.  A request's block table names its pages in order; token t of the request is row
table[t // page] * page + t % page.

* ``plan``     block tables and slot maps of one scheduler step from the requests' lengths: pages of finished requests go back to the
               pool, new tokens get pages from it, every new token its row (``ops.page_plan``)
* ``store``    K and V vectors of new tokens into the rows of a slot map, and those rows back as vectors, as an export or another
               attention reads them (``ops.paged_append``, ``ops.paged_read``)
* ``decode``   attention of one query token per request over its pages (``ops.paged_decode_attention``)
* ``prefill``  causal attention of several new tokens per request, a ragged batch, over earlier and new tokens
               (``ops.paged_prefill_attention``)

`own` chooses between the library's calls and the plain forms, which are elementary torch operations in 32 bits (rotations and
quantiser decisions, which lie next to borders, in 64).  Values: K, V and queries ~ N(0, 1), as after a model's norms; cached codes are
those of normal vectors.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

D = 128
CENTROIDS = {4: [0.01135, 0.03432, 0.05806, 0.08330, 0.11099, 0.14304, 0.18293, 0.24155], 2: [0.04003, 0.13351]}
BOUNDS = {4: [0.02284, 0.04619, 0.07068, 0.09715, 0.12701, 0.16299, 0.21224], 2: [0.08677]}


def _case(op, name=None, **kw):
    c = dict(op=op, **kw)
    return dict(c, name=name) if name else c


def listed():
    return [
        # every decode step of a rollout batch: a token for each running request, a few of which have just ended
        _case("plan", "plan-decode-256", seqs=256, page=64, context=4096, new=1, finished=5),
        # a step that starts prompts beside running requests: slot maps of up to 65536 tokens
        _case("plan", "plan-prompts-64x2048", seqs=64, page=32, context=2019, new=2048, finished=7),
        # the new tokens of a decode step
        _case("store", "store-4bit-64", bits=4, kv_heads=8, tokens=64, page=64, fused=True),
        # a small prompt batch of odd length, 2-bit, four KV heads
        _case("store", "store-2bit-1777", bits=2, kv_heads=4, tokens=1777, page=32, fused=False),
        # a chunk of prompts
        _case("store", "store-4bit-8192", bits=4, kv_heads=8, tokens=8192, page=64, fused=True),
        # four rollouts of one short prompt: the smallest batched call
        _case("decode", "decode-4bit-4x612", bits=4, heads=16, kv_heads=8, seqs=4, longest=612, shortest=612, page=64),
        # a rollout batch at context 4096
        _case("decode", "decode-4bit-64x4096", bits=4, heads=16, kv_heads=8, seqs=64, longest=4096, shortest=4096, page=64),
        # the larger model, long contexts, 2-bit
        _case("decode", "decode-2bit-32x8192", bits=2, heads=32, kv_heads=8, seqs=32, longest=8192, shortest=8192, page=128),
        # a continuous batch of very different lengths, some of its places empty
        _case("decode", "decode-4bit-ragged-128", bits=4, heads=32, kv_heads=8, seqs=128, longest=16384, shortest=0, page=32),
        # prompts without earlier tokens
        _case("prefill", "prefill-4bit-8x512", bits=4, heads=16, kv_heads=8, seqs=8, context=0, new=512, shortest_new=512, page=64),
        # chunks of long prompts: 1024 new tokens behind 8192
        _case("prefill", "prefill-4bit-4x1024+8192", bits=4, heads=32, kv_heads=8, seqs=4, context=8192, new=1024, shortest_new=1000, page=64),
        # drafted tokens of running requests, checked in one pass
        _case("prefill", "prefill-2bit-32x5+4000", bits=2, heads=32, kv_heads=8, seqs=32, context=4000, new=5, shortest_new=1, page=128),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


LAYOUTS = [(16, 8), (32, 8), (16, 4), (32, 4), (8, 8), (40, 8), (14, 2), (8, 1)]


def draw(rng):
    op = rng.choice(["plan", "store", "decode", "decode", "prefill", "prefill"])
    page = rng.choice([32, 64, 128, 256])
    if op == "plan":
        seqs, new = _log(rng, 1, 1024), rng.choice([1, 1, _log(rng, 2, 2048)])
        return _case(op, seqs=seqs, page=page, context=_log(rng, 16, 8192), new=min(new, 131072 // seqs), finished=rng.randint(0, min(8, seqs)))
    bits = rng.choice([4, 4, 2])
    if op == "store":
        return _case(op, bits=bits, kv_heads=rng.choice([8, 8, 4, 2, 1]), tokens=_log(rng, 1, 8192), page=page, fused=rng.random() < 0.5)
    heads, kv_heads = rng.choice(LAYOUTS)
    if op == "decode":
        longest = _log(rng, 1, 16384)
        seqs = _log(rng, 1, max(1, min(256, 131072 * 8 // (longest * kv_heads))))
        return _case(op, bits=bits, heads=heads, kv_heads=kv_heads, seqs=seqs, longest=longest, shortest=rng.choice([longest, longest // 2, 0]), page=page)
    new, context = _log(rng, 1, 2048), rng.choice([0, _log(rng, 1, 12000)])
    most = max(1, min(64, 4 * 1024 * 9216 * 32 // (new * (new + context) * heads)))
    return _case(op, bits=bits, heads=heads, kv_heads=kv_heads, seqs=_log(rng, 1, most), context=context, new=new, shortest_new=rng.choice([new, max(1, new // 2), 0]), page=page)


# ---- inputs ---------------------------------------------------------------------------------------------------------------------------
def _rotation(gen):
    q, _ = torch.linalg.qr(torch.randn(D, D, generator=gen, device="cuda", dtype=torch.float64))
    return q.to(torch.float16).contiguous()


def _codes(gen, rows, kv_heads, bits):
    """Packed codes and norms of `rows` tokens of normal vectors."""
    bounds = torch.tensor([-b for b in reversed(BOUNDS[bits])] + [0.0] + BOUNDS[bits], device="cuda") * math.sqrt(D)
    per = 8 // bits
    codes = torch.bucketize(torch.randn(rows, kv_heads * D, generator=gen, device="cuda"), bounds, out_int32=True).to(torch.uint8)
    codes = codes.view(rows, kv_heads * D // per, per)
    packed = codes[:, :, 0].clone()
    for j in range(1, per):
        packed |= codes[:, :, j] << (bits * j)
    norms = (math.sqrt(D) * (1.0 + 0.0625 * torch.randn(rows, kv_heads, generator=gen, device="cuda"))).to(torch.float16)
    return packed, norms


def _tables(rs, lens, width, page):
    """A pool's pages in no order, handed to the requests in turn: table [seqs][width], the pool's size, the pages left over."""
    need = -(-lens // page)
    total = int(need.sum())
    spare = total // 16 + 4
    order = rs.permutation(total + spare).astype(np.int32)
    table = np.zeros((len(lens), width), np.int32)
    at = 0
    for g, n in enumerate(need):
        table[g, :n] = order[at:at + n]
        at += n
    return table, total + spare, order[at:]


def _lengths(case):
    """(tokens held, new tokens, ended) of each request: the same for every seed, as the outputs' shapes go by them."""
    rs, G = np.random.RandomState(case["seqs"] + case["page"]), case["seqs"]
    ended = np.zeros(G, np.uint8)
    if case["op"] == "decode":
        held = rs.randint(case["shortest"], case["longest"] + 1, G)
        held[0] = case["longest"]
        return np.maximum(held - 1, 0), np.minimum(held, 1), ended
    if case["op"] == "prefill":
        new, held = rs.randint(case["shortest_new"], case["new"] + 1, G), rs.randint(case["context"] // 2, case["context"] + 1, G)
        new[0], held[0] = case["new"], case["context"]
        return held, new, ended
    ended[rs.choice(G, min(G, case["finished"]), replace=False)] = 1
    held = rs.randint(0, case["context"] + 1, G)
    new = np.ones(G, np.int64) if case["new"] == 1 else rs.randint(0, case["new"] + 1, G)
    return held, np.where(ended, 0, new), ended


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rs = np.random.RandomState(seed % (1 << 31))
    op, page = case["op"], case["page"]
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    if op == "plan":
        G = case["seqs"]
        context, new, ended = _lengths(case)
        context, new = context.astype(np.int32), new.astype(np.int32)
        width = -(-(case["context"] + case["new"]) // page)
        table, pages, free = _tables(rs, context, width, page)
        want = int((-(-(context + new) // page) + context // -page).sum())
        more = np.arange(pages, pages + max(0, want - len(free) + 2), dtype=np.int32)
        stack = np.zeros(pages + len(more), np.int32)
        stack[:len(free) + len(more)] = np.concatenate([free, more])
        T = int(new.sum()) + 3  # (a buffer a little longer than the tokens)
        s = dict(table=dev(table), free=dev(stack), count=dev(np.array([len(free) + len(more)], np.int32)), context=dev(context), new=dev(new),
                 finished=dev(ended))
        for name, n, t in (("count_out", 1, torch.int32), ("lens", G, torch.int32), ("start", G + 1, torch.int32), ("slots", T, torch.int64), ("positions", T, torch.int32)):
            s[name] = torch.empty(n, dtype=t, device="cuda")
        return dict(case=case, **s)
    bits, Hkv = case["bits"], case["kv_heads"]
    R = _rotation(gen)
    if op == "store":
        T = case["tokens"]
        lens = np.array([T - T // 3, T // 3 + 1])
        table, pages, _ = _tables(rs, lens, -(-int(lens.max()) // page), page)
        t = np.arange(int(lens[0]))
        slots = np.concatenate([table[g, t[:n] // page].astype(np.int64) * page + t[:n] % page for g, n in enumerate(lens)])[:T]
        if T > 8:
            slots[rs.choice(T, T // 64 + 1, replace=False)] = -1  # (padding)
        codes = [_codes(gen, pages * page, Hkv, bits) for _ in range(2)]
        if case["fused"]:  # a projection's output: queries, keys and values of a token side by side
            qkv = torch.randn(T, 4 * Hkv * D, generator=gen, device="cuda").to(torch.float16)
            k, v = qkv[:, 2 * Hkv * D:3 * Hkv * D], qkv[:, 3 * Hkv * D:]
        else:
            k, v = (torch.randn(T, Hkv * D, generator=gen, device="cuda").to(torch.float16) for _ in range(2))
        return dict(case=case, R=R, k=k, v=v, slots=dev(slots), ck=codes[0][0], kn=codes[0][1], cv=codes[1][0], vn=codes[1][1],
                    k_out=torch.empty(T, Hkv * D, dtype=torch.float16, device="cuda"), v_out=torch.empty(T, Hkv * D, dtype=torch.float16, device="cuda"))
    G, H = case["seqs"], case["heads"]
    held, new, _ = _lengths(case)
    lens = held + new
    start = np.arange(G + 1) if op == "decode" else np.concatenate([[0], np.cumsum(new)])  # (an empty place of a decode batch has a query too)
    table, pages, _ = _tables(rs, lens, -(-int(lens.max()) // page) + 1, page)
    (ck, kn), (cv, vn) = (_codes(gen, pages * page, Hkv, bits) for _ in range(2))
    T = int(start[-1])
    q = torch.randn(T, H * D, generator=gen, device="cuda").to(torch.float16)
    return dict(case=case, R=R, q=q, out=torch.empty_like(q), ck=ck, kn=kn, cv=cv, vn=vn, table=dev(table), lens=dev(lens.astype(np.int32)),
                start=dev(start.astype(np.int32)), longest=int(lens.max()), most_new=int(new.max()), work={})


# ---- the plain forms ------------------------------------------------------------------------------------------------------------------
def _values(codes, bits):
    """Packed bytes [..., n] as 32-bit centroids [..., n * codes per byte]."""
    half = CENTROIDS[bits]
    c = torch.tensor([-x for x in reversed(half)] + half, device=codes.device)
    byte = torch.arange(256, device=codes.device)
    table = torch.stack([c[(byte >> s) & ((1 << bits) - 1)] for s in range(0, 8, bits)], dim=-1)
    return table[codes.int()].flatten(-2)


def _plain_plan(s):
    page, table = s["case"]["page"], s["table"]
    G, W = table.shape
    col = torch.arange(W, device="cuda")
    old = torch.where(s["context"] < 0, ~s["context"], s["context"]).long()
    ended = s["finished"] != 0
    back = ended[:, None] & (col < ((old + page - 1) // page)[:, None])
    released = table[back]
    count = s["count"].long()
    have = count + released.numel()
    s["free"][count + torch.arange(released.numel(), device="cuda")] = released
    context = torch.where(ended, 0, old)
    new = s["new"].long().clamp(min=0)
    first, last = (context + page - 1) // page, (context + new + page - 1) // page
    fits = context + new <= W * page
    need = torch.where(fits, last - first, 0)
    upto, tokens = need.cumsum(0), new.cumsum(0)
    T = s["slots"].numel()
    admitted = fits & ((new == 0) | ((tokens <= T) & ((need == 0) | (upto <= have))))
    s["count_out"].copy_(have - torch.where(admitted, need, 0).sum())
    fresh = admitted[:, None] & (col >= first[:, None]) & (col < last[:, None])
    k = (upto - need)[:, None] + col - first[:, None]
    table[fresh] = s["free"][(have - 1 - k)[fresh]]
    s["lens"].copy_(torch.where(admitted, context + new, ~context))
    s["start"][0] = 0
    s["start"][1:] = tokens.clamp(max=T)
    t = torch.arange(T, device="cuda")
    g = torch.searchsorted(tokens, t, right=True)
    real = g < G
    g = g.clamp(max=G - 1)
    real = real & admitted[g]
    pos = torch.where(real, context[g] + t - (tokens - new)[g], -1)
    s["positions"].copy_(pos)
    s["slots"].copy_(torch.where(real, table[g, (pos.clamp(min=0) // page)].long() * page + pos % page, -1))


def _plain_store(s):
    bits, Hkv = s["case"]["bits"], s["case"]["kv_heads"]
    R = s["R"].double()
    bounds = torch.tensor([-b for b in reversed(BOUNDS[bits])] + [0.0] + BOUNDS[bits], device="cuda", dtype=torch.float64)
    keep = s["slots"] >= 0
    rows = s["slots"][keep]

    def write(x, codes, norms):
        v = x[keep].double().view(-1, Hkv, D)
        n = (v.square().sum(-1, keepdim=True) + 1e-12).sqrt()
        code = torch.bucketize((v / n) @ R.T, bounds, right=True)  # (how many bounds a coordinate has reached)
        per = 8 // bits
        byte = (code.view(-1, Hkv * D // per, per) << (bits * torch.arange(per, device="cuda"))).sum(-1)
        codes[rows] = byte.to(torch.uint8)
        norms[rows] = n[..., 0].to(torch.float16)

    def read(codes, norms, out):
        x = _values(codes[rows], bits).view(-1, Hkv, D) * norms[rows].float()[..., None]
        out.zero_()
        out[keep] = (x @ s["R"].float()).to(torch.float16).view(-1, Hkv * D)

    write(s["k"], s["ck"], s["kn"])
    write(s["v"], s["cv"], s["vn"])
    read(s["ck"], s["kn"], s["k_out"])
    read(s["cv"], s["vn"], s["v_out"])


def _plain_attention(s):
    c = s["case"]
    bits, page, H, Hkv, G, L, N = c["bits"], c["page"], c["heads"], c["kv_heads"], c["seqs"], s["longest"], s["most_new"]
    t = torch.arange(L, device="cuda")
    rows = s["table"].long()[:, t // page] * page + t % page
    lens, start = s["lens"].long(), s["start"].long()
    first = lens - (start[1:] - start[:-1])  # position of a request's first query
    i = torch.arange(N, device="cuda")
    there = i < (start[1:] - start[:-1])[:, None]
    at = torch.where(there, start[:-1, None] + i, 0)
    R = s["R"].float()
    q = (s["q"].float()[at].view(G, N, Hkv, H // Hkv, D) @ R.T).permute(0, 2, 1, 3, 4).reshape(G, Hkv, N * (H // Hkv), D)
    k = _values(s["ck"][rows], bits).view(G, L, Hkv, D).transpose(1, 2)
    x = (q @ k.transpose(2, 3) * (s["kn"][rows].float().transpose(1, 2)[:, :, None] / math.sqrt(D))).view(G, Hkv, N, H // Hkv, L)
    seen = t <= (first[:, None] + i)[:, None, :, None, None]
    seen = seen & (t < lens[:, None, None, None, None])
    x = torch.where(seen, x, -math.inf)
    top = x.amax(-1, keepdim=True)
    w = torch.where(seen, (x - top).exp(), 0.0)
    z = w.sum(-1, keepdim=True)
    w = w * (s["vn"][rows].float().transpose(1, 2)[:, :, None, None])
    v = _values(s["cv"][rows], bits).view(G, L, Hkv, D).transpose(1, 2)
    o = (w.reshape(G, Hkv, N * (H // Hkv), L) @ v).view(G, Hkv, N, H // Hkv, D) / torch.where(z > 0, z, 1.0)
    o = (o @ R).permute(0, 2, 1, 3, 4).reshape(G, N, H * D)
    s["out"][at[there]] = o[there].to(torch.float16)


def run(s):
    c = s["case"]
    op = c["op"]
    if op == "plan":
        if own:
            from triebwerk_b200 import ops
            ops.page_plan(s["table"], s["free"], s["count"], s["count_out"], s["context"], s["new"], s["finished"], c["page"], s["lens"], s["start"],
                          s["slots"], s["positions"])
        else:
            _plain_plan(s)
        return {k: s[k] for k in ("table", "free", "count_out", "lens", "start", "slots", "positions")}
    if op == "store":
        if own:
            from triebwerk_b200 import ops
            ops.paged_append(s["ck"], s["kn"], s["cv"], s["vn"], s["k"], s["v"], s["R"], s["slots"], c["kv_heads"], c["bits"])
            ops.paged_read(s["k_out"], s["v_out"], s["ck"], s["kn"], s["cv"], s["vn"], s["R"], s["slots"], c["kv_heads"], c["bits"])
        else:
            _plain_store(s)
        return {"k": s["k_out"], "v": s["v_out"]}
    if own:
        from triebwerk_b200 import ops
        if "ws" not in s["work"]:  # (a program's workspace, kept from call to call)
            s["work"]["ws"] = ops.paged_workspace(s["q"].shape[0], c["seqs"], c["heads"])
        args = (s["out"], s["q"], s["ck"], s["cv"], s["kn"], s["vn"], s["R"], s["table"], s["lens"])
        if op == "decode":
            ops.paged_decode_attention(*args, c["page"], c["heads"], c["kv_heads"], c["bits"], s["work"]["ws"])
        else:
            ops.paged_prefill_attention(*args, s["start"], c["page"], c["heads"], c["kv_heads"], c["bits"], s["work"]["ws"])
    else:
        _plain_attention(s)
    return {"out": s["out"]}


def work(case):
    c = case
    if c["op"] == "plan":  # (lengths, flags and starts; slot and position of a token; the pages that change hands, read here and written there)
        held, new, ended = _lengths(c)
        pages = (-(-(held + new) // c["page"]) + held // -c["page"])[ended == 0].sum() + (-(-held // c["page"]))[ended != 0].sum()
        return {"bytes": int(17 * c["seqs"] + 12 * (new.sum() + 3) + 8 * pages), "flops": 0}
    row = c["kv_heads"] * (D * c["bits"] // 8 + 2)  # bytes of a token's K or V in the cache
    if c["op"] == "store":
        T = c["tokens"]
        return {"bytes": 2 * T * (2 * 2 * c["kv_heads"] * D + 2 * row) + 2 * 8 * T + 4 * D * D, "flops": 2 * 2 * 2 * T * c["kv_heads"] * D * D}
    held, new, _ = _lengths(c)
    tokens, pairs = int((held + new)[new > 0].sum()), int((new * held + new * (new + 1) // 2).sum())
    queries = c["seqs"] if c["op"] == "decode" else int(new.sum())
    return {"bytes": 2 * tokens * row + 2 * 2 * queries * c["heads"] * D + 2 * D * D, "flops": 4 * pairs * c["heads"] * D + 4 * queries * c["heads"] * D * D}


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------------------------
def exact(case, seed):
    if case["op"] == "plan":
        return None  # (whole numbers)
    s = prepare(case, seed)
    bits, Hkv = case["bits"], case["kv_heads"]
    R = s["R"].double()
    up = CENTROIDS[bits]
    cent = torch.tensor([-x for x in up[::-1]] + up, device="cuda", dtype=torch.float64)

    def vectors(codes, norms):  # rows of the cache as the vectors that they stand for, [rows][Hkv][128]
        c = torch.stack([(codes >> sh) & (2 ** bits - 1) for sh in range(0, 8, bits)], -1).reshape(codes.shape[0], Hkv, D)
        return torch.einsum("rhk,kd->rhd", cent[c.long()] * norms.double()[:, :, None], R)

    if case["op"] == "store":
        edge = torch.tensor([-x for x in BOUNDS[bits][::-1]] + [0.0] + BOUNDS[bits], device="cuda", dtype=torch.float64)
        out = {}
        for name in ("k", "v"):
            x = s[name].double().reshape(-1, Hkv, D)
            n = torch.sqrt(torch.einsum("thd,thd->th", x, x) + 1e-12)
            y = torch.einsum("thd,kd->thk", x, R) / n[:, :, None]
            code = sum((y >= e).long() for e in edge)
            back = torch.einsum("thk,kd->thd", cent[code] * n.to(torch.float16).double()[:, :, None], R)
            out[name] = torch.where(s["slots"][:, None] >= 0, back.reshape(-1, Hkv * D), 0.0)
        return out
    H, page = case["heads"], case["page"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lens, start, table = s["lens"].tolist(), s["start"].tolist(), s["table"].long()
    for g, n in enumerate(lens):
        a, b = start[g], start[g + 1]
        if n == 0 or a == b:
            continue
        rows = (table[g, :-(-n // page), None] * page + torch.arange(page, device="cuda")).reshape(-1)[:n]
        q = s["q"][a:b].double().view(b - a, H, D)
        k, v = vectors(s["ck"][rows], s["kn"][rows]), vectors(s["cv"][rows], s["vn"][rows])
        hidden = torch.arange(n, device="cuda")[None, :] > (n - (b - a) + torch.arange(b - a, device="cuda"))[:, None]
        for h in range(Hkv):
            qh = q[:, h * (H // Hkv):(h + 1) * (H // Hkv)]
            x = torch.einsum("qhd,kd->hqk", qh, k[:, h]) / math.sqrt(D)
            p = torch.softmax(x.masked_fill(hidden, -math.inf), -1)
            out[a:b, h * (H // Hkv) * D:(h + 1) * (H // Hkv) * D] = torch.einsum("hqk,kd->qhd", p, v[:, h]).reshape(b - a, -1)
    return {"out": out}
