"""Paged attention over the whole range of norms, with norms that are not finite among the new tokens, and with many query heads per KV head."""
import numpy as np
import pytest
import torch

from tests import paged_util as pu

pytestmark = pytest.mark.gpu
gu = pytest.importorskip("tests.gpu_util")
from tests.test_paged_gpu import attention_inputs, check_prefill, i32, no_status  # noqa: E402,F401
from triebwerk_b200 import ops  # noqa: E402


def spread(rng, shape, low, high):
    """Norms whose logarithms are spread evenly."""
    return torch.from_numpy(np.exp(rng.uniform(np.log(low), np.log(high), shape)).astype(np.float16)).cuda()


def attention(q, ck, cv, kn, vn, R, table, lens, start, page, H, Hkv, bits):
    """pu.attention with a bound for norms of any size: (out, tolerance [T, H] in 2-norm).

    The same roundings, each relative and by a variance of at most EPS^2 / 3, but their effect in full.  With w the weights, a score's error d_t moves
    the weights' sum too: out = sum w_t v_t changes by sum_t w_t d_t (v_t - out), where v_t alone, as pu.attention has it, is enough only while no token's v is
    far longer than another's.  A weight's (times its norm) and a V centroid's rounding move it by w_t v_t EPS each.  Six roots of the variances' sum, and
    2 EPS |out| as there.
    fp16 numbers below 2^-14 are off by 2^-25 however small they are: weights times norms (each of n moves the result by 2^-25 |c|, c the row's centroids,
    next to a sum of weights of at least 1) or weights (2^-25 |v| each), centroids times norms (2^-25 a coordinate under weights whose sum is 1:
    2^-25 sqrt(128)), and results before and behind R (as much each)."""
    T, EPS = q.shape[0], pu.EPS
    out = torch.zeros(T, H, 128, dtype=torch.float64, device="cuda")
    tol = torch.zeros(T, H, dtype=torch.float64, device="cuda")
    c = torch.tensor([-x for x in reversed(pu.CENT[bits])] + pu.CENT[bits], dtype=torch.float64, device="cuda")
    Rd = R.double()
    for g, n in enumerate(lens):
        a, b = start[g], start[g + 1]
        if n <= 0 or a == b:
            continue
        rows = pu.rows_of(table[g], n, page)
        k, v = (c[torch.stack([(codes[rows] >> s) & ((1 << bits) - 1) for s in range(0, 8, bits)], -1).reshape(n, Hkv, 128).long()] * norms[rows].double()[..., None]
                for codes, norms in ((ck, kn), (cv, vn)))
        qr = q[a:b].double().view(b - a, Hkv, H // Hkv, 128) @ Rd.T / 128**0.5
        x = torch.einsum("qhgd,khd->hgqk", qr, k)
        pos = n - (b - a) + torch.arange(b - a, device="cuda")
        w = torch.softmax(x.masked_fill(torch.arange(n, device="cuda")[None] > pos[:, None], -float("inf")), -1).nan_to_num(0.0)
        o = torch.einsum("hgqk,khd->qhgd", w, v)
        v2 = v.square().sum(-1).T[:, None, None]  # [Hkv, 1, 1, n]
        apart = (v2 - 2 * torch.einsum("qhgd,khd->hgqk", o, v) + o.square().sum(-1).permute(1, 2, 0)[..., None]).clamp(min=0.0)  # |v_t - out|^2
        moved = w.square() * EPS**2 * 2 / 3 * (torch.einsum("qhgd,khd->hgqk", qr.square(), k.square()) * apart + v2)
        tol[a:b] = (6 * moved.sum(-1).sqrt() + n * 2.0**-25 * v2.amax(-1).sqrt()).permute(2, 0, 1).reshape(b - a, H)
        out[a:b] = (o @ Rd).reshape(b - a, H, 128)
    longest = max(pu.CENT[bits]) * 128**0.5  # of a row of centroids
    return out.view(T, H * 128), tol + 2 * EPS * out.norm(dim=-1) + 2.0**-25 * (max(lens) * longest + 3 * 128**0.5)


def check_spread(lens, new, H, Hkv, bits, seed, wide_k, decode=False):
    """Norms from 0.01 to 60000 next to each other, of V (K's as far as scores stay below a hundred) or, with small queries, of both."""
    rng = np.random.default_rng(seed)
    start = [0] + np.cumsum(new).tolist()
    table, q, out, ck, cv, kn, vn, R, _ = attention_inputs(rng, lens, H, Hkv, bits, 32, T=start[-1])
    held = torch.cat([pu.rows_of(table[g], n, 32) for g, n in enumerate(lens) if n > 0])
    vn[held] = spread(rng, (len(held), Hkv), 1e-2, 6e4)
    kn[held] = spread(rng, (len(held), Hkv), 1e-2, 6e4 if wide_k else 30.0)
    if wide_k:
        q *= 0.01
    ws = ops.paged_workspace(start[-1], len(lens), H)
    if decode:
        ops.paged_decode_attention(out, q, ck, cv, kn, vn, R, table, i32(lens), 32, H, Hkv, bits, ws)
    else:
        ops.paged_prefill_attention(out, q, ck, cv, kn, vn, R, table, i32(lens), i32(start), 32, H, Hkv, bits, ws)
    torch.cuda.synchronize()
    pu.assert_attention(out, attention(q, ck, cv, kn, vn, R, table, lens, start, 32, H, Hkv, bits), f"{bits}-bit {H}/{Hkv}")


@pytest.mark.parametrize("bits", [4, 2])
@pytest.mark.parametrize("wide_k", [False, True])
@pytest.mark.parametrize("H, Hkv, lens, new", [
    (32, 8, [700, 41, 5, 333], [5, 1, 5, 8]),     # few rows: one to four blocks of them
    (32, 8, [900] * 6, [5] * 6), (16, 8, [300, 64], [3, 4]),
    (32, 8, [5000], [4]),                         # ... cut along the context
    (14, 2, [6000], [40]),                        # many rows, cut along the context
    (16, 8, [300, 420], [300, 70]),               # one block a CTA
    (16, 8, [1500, 900, 700, 800] * 4, [1000, 700, 700, 600] * 4),  # two
])
def test_prefill_norms_of_every_size(H, Hkv, lens, new, bits, wide_k):
    check_spread(lens, new, H, Hkv, bits, H + len(lens) + lens[0], wide_k)


@pytest.mark.parametrize("bits", [4, 2])
@pytest.mark.parametrize("wide_k", [False, True])
@pytest.mark.parametrize("H, Hkv, lens", [(16, 8, [600, 1, 33, 70]), (40, 8, [600, 90, 33]), (32, 8, [3000] * 40), (16, 4, [3000] * 70)])
def test_decode_norms_of_every_size(H, Hkv, lens, bits, wide_k):
    check_spread(lens, [1] * len(lens), H, Hkv, bits, H + len(lens), wide_k, decode=True)


@pytest.mark.parametrize("bits", [4, 2])
@pytest.mark.parametrize("H, Hkv, lens, new", [(16, 8, [700, 700], [5, 5]), (32, 8, [9000, 90], [5, 3]), (14, 2, [6000], [40]), (32, 4, [5000], [60]), (16, 8, [900] * 20, [600] * 20)])
@pytest.mark.parametrize("name, value", [("v", float("nan")), ("v", float("inf")), ("v", -float("inf")), ("k", float("nan")), ("k", float("inf")), ("k", -float("inf"))])
def test_prefill_a_norm_that_is_not_finite_among_the_new_tokens(H, Hkv, lens, new, bits, name, value):
    # queries in front of the token, other requests and other heads stay as they are; those that see a NaN, or an infinite value, are not finite
    rng = np.random.default_rng(lens[0] + bits)
    start, grp, head = [0] + np.cumsum(new).tolist(), H // Hkv, Hkv - 1
    table, q, out, ck, cv, kn, vn, R, _ = attention_inputs(rng, lens, H, Hkv, bits, 32, T=start[-1])
    first = new[0] // 2  # of the queries that see it
    want = pu.attention(q, ck, cv, kn, vn, R, table, lens, start, 32, H, Hkv, bits)
    at = pu.rows_of(table[0], lens[0], 32)[lens[0] - new[0] + first]
    (vn if name == "v" else kn)[at, head] = value
    ws = ops.paged_workspace(start[-1], len(lens), H)
    ops.paged_prefill_attention(out, q, ck, cv, kn, vn, R, table, i32(lens), i32(start), 32, H, Hkv, bits, ws)
    torch.cuda.synchronize()
    sees = torch.zeros(start[-1], H, dtype=torch.bool, device="cuda")
    sees[first:new[0], head * grp:] = True
    finite = out.isfinite().view(start[-1], H, 128).all(-1)
    assert finite[~sees].all()
    if name == "v" or value != value:
        assert not finite[sees].any()
    hidden = torch.where(sees[..., None], want[0].view(-1, H, 128).half(), out.view(-1, H, 128)).view(out.shape)
    pu.assert_attention(hidden, (want[0], torch.where(sees, float("inf"), want[1])))


@pytest.mark.parametrize("bits", [4, 2])
@pytest.mark.parametrize("H, Hkv", [(20, 1), (32, 1), (33, 1), (40, 1), (100, 1), (128, 1), (256, 2), (96, 3)])
def test_prefill_many_query_heads(H, Hkv, bits):
    check_prefill([1, 0, 5, 40, 300, 71, 90, 1000], [1, 0, 5, 33, 1, 70, 0, 9], H, Hkv, bits, 32, H + bits)
    check_prefill([77], [77], H, Hkv, bits, 64, 1, tail=0)                       # one request
    check_prefill([1], [1], H, Hkv, bits, 64, 2, tail=0)
    check_prefill([5000], [1], H, Hkv, bits, 64, 3, tail=1)                      # cut along the context
    check_prefill([4000, 3], [3, 2], H, Hkv, bits, 64, 4)
    check_prefill([700, 200, 333, 12], [300, 200, 31, 12], H, Hkv, bits, 128, 5)  # two blocks a CTA
    check_prefill([900 + 17 * g for g in range(40)], [1] * 40, H, Hkv, bits, 32, 6, tail=0)


@pytest.mark.parametrize("G, form", [(4, "streaming"), (5, "cluster"), (40, "cluster")])
def test_decode_more_tiles_than_can_be_numbered(G, form):
    # Tables with room for 2^26 - 2048 tiles a request, of shared pages: 5 requests could pass 2^28 and 33 of them 2^31, which the streaming form's tile
    # numbers do not hold.  The cluster form, which has none, writes nothing to the workspace.
    rng = np.random.default_rng(G)
    page, width, H, Hkv, bits = 65536, 32767, 16, 8, 2
    (ck, kn), (cv, vn) = (pu.random_cache(rng, page, Hkv, bits) for _ in range(2))
    lens = rng.integers(0, 3000, G).tolist()
    table = torch.zeros(G, width, dtype=torch.int32, device="cuda")
    q = torch.from_numpy(rng.standard_normal((G, H * 128)).astype(np.float16)).cuda()
    out, R, ws = torch.empty_like(q), pu.rotation(5).cuda(), ops.paged_workspace(G, G, H)
    ws.fill_(77)
    ops.paged_decode_attention(out, q, ck, cv, kn, vn, R, table, i32(lens), page, H, Hkv, bits, ws)
    torch.cuda.synchronize()
    assert (form == "cluster") == bool((ws == 77).all())
    pu.assert_attention(out, pu.attention(q, ck, cv, kn, vn, R, table, lens, list(range(G + 1)), page, H, Hkv, bits))


@pytest.mark.parametrize("new", [1, 7, 60])
def test_results_between_the_rows_of_queries(new):
    # one array of four columns: queries in the first (every row), results in the second and fourth in turn, rows half as far apart
    rng = np.random.default_rng(new)
    G, H, Hkv, page = 5, 16, 8, 32
    W, T, lens, start = H * 128, G * new, [100 + 30 * g for g in range(G)], [new * g for g in range(G + 1)]
    table, q, _, ck, cv, kn, vn, R, _ = attention_inputs(rng, lens, H, Hkv, 4, page, T=T)
    whole = torch.full((T, 4 * W), 7.0, dtype=torch.float16, device="cuda")
    mine, out = whole[:, :W], whole.view(2 * T, 2 * W)[:T, W:]
    mine.copy_(q)
    apart = torch.empty(T, W, dtype=torch.float16, device="cuda")
    ws = ops.paged_workspace(T, G, H)
    for a, o in ((q, apart), (mine, out)):
        ops.paged_prefill_attention(o, a, ck, cv, kn, vn, R, table, i32(lens), i32(start), page, H, Hkv, 4, ws)
        if new == 1:
            ops.paged_decode_attention(o, a, ck, cv, kn, vn, R, table, i32(lens), page, H, Hkv, 4, ws)
    torch.cuda.synchronize()
    assert torch.equal(out, apart) and torch.equal(mine, q) and (whole[:, 2 * W:3 * W] == 7).all()


# ---- one long request among small ones ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("bits", [4, 2])
@pytest.mark.parametrize("H, Hkv, small, chunk, past, at", [
    (32, 8, 63, 64, 9000, 0), (32, 8, 63, 65, 9000, 63),   # (the second: tokens in a multiple of the requests)
    (32, 8, 15, 200, 5000, 7), (16, 8, 31, 100, 3000, 30), (4, 1, 700, 64, 6000, 650), (14, 2, 20, 90, 2500, 3), (16, 1, 5, 40, 4000, 5), (32, 8, 1, 64, 6000, 1)])
def test_prefill_a_chunk_beside_single_tokens(H, Hkv, small, chunk, past, at, bits):
    rng = np.random.default_rng(small + chunk)
    lens, new = rng.integers(0, 700, small).tolist(), [1] * small
    lens.insert(at, past + chunk)
    new.insert(at, chunk)
    check_prefill(lens, new, H, Hkv, bits, 64, small, tail=0)
    for g in range(0, small, 5):
        if g != at:
            new[g] = (0, 3, 2)[g % 3]
    check_prefill(lens, new, H, Hkv, bits, 64, small + 1, tail=5)
    lens[at] = chunk // 2  # more queries than tokens
    check_prefill(lens, new, H, Hkv, bits, 64, small + 2, tail=1)


@pytest.mark.parametrize("bits", [4, 2])
@pytest.mark.parametrize("H, Hkv, new", [(32, 8, [9 + g % 12 for g in range(16)]), (16, 8, list(range(17, 41, 3))), (32, 8, [20 + 5 * g for g in range(8)]), (32, 8, [3, 5, 8, 9, 12, 20, 4, 6, 2, 1, 15, 3])])
def test_prefill_requests_of_a_few_to_a_few_dozen_tokens(H, Hkv, new, bits):
    # whole and cut blocks, of one launch
    check_prefill([n + 2600 + 100 * g for g, n in enumerate(new)], new, H, Hkv, bits, 32, len(new))
    check_prefill([n + 30 * g for g, n in enumerate(new)], new, H, Hkv, bits, 32, len(new), tail=0)


def test_prefill_captured_batches_of_every_kind():
    # one graph, whose replays hand the same 96 query rows out to the requests in other ways: the parts of a block follow
    rng = np.random.default_rng(3)
    T, G, H, Hkv, bits, page = 96, 20, 32, 8, 4, 32
    lens = [3000 + 50 * g for g in range(G)]
    table, q, out, ck, cv, kn, vn, R, _ = attention_inputs(rng, lens, H, Hkv, bits, page, T=T)
    d, st, ws = i32(lens), i32(np.zeros(G + 1)), ops.paged_workspace(T, G, H)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        ops.paged_prefill_attention(out, q, ck, cv, kn, vn, R, table, d, st, page, H, Hkv, bits, ws)
    for new in ([77] + [1] * 19, [1] * 20, [5] * 19 + [1], [0] * 19 + [96], [9] * 10 + [0] * 10, [0] * 20, [1] * 10 + [43] * 2 + [0] * 8, [48, 48] + [0] * 18, [40, 1, 0] * 2 + [0] * 14):
        start = [0] + np.cumsum(new).tolist()
        st.copy_(i32(start))
        ws.fill_(255)  # (nothing is kept in it)
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        want = pu.attention(q, ck, cv, kn, vn, R, table, lens, start, page, H, Hkv, bits)
        pu.assert_attention(out[:start[-1]], (want[0][:start[-1]], want[1][:start[-1]]), str(new))
        assert (out[start[-1]:] == 7).all()


@pytest.mark.parametrize("chunk", [64, 65])
def test_single_tokens_do_not_slow_a_chunk_down(chunk):
    # (Its context is cut along the SMs that idle, with single tokens beside it as alone; uncut beside 63 it took 7 times as long as alone, cut 2.4 times, theirs
    # included.  The fastest of some rounds, so that other work on the machine does not count.)
    def us(lens, new, H=32, Hkv=8, bits=4, page=64):
        rng = np.random.default_rng(0)
        start = [0] + np.cumsum(new).tolist()
        table, q, out, ck, cv, kn, vn, R, _ = attention_inputs(rng, lens, H, Hkv, bits, page, T=start[-1])
        d, st, ws = i32(lens), i32(start), ops.paged_workspace(start[-1], len(lens), H)
        best = []
        for _ in range(8):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            for _ in range(10):
                ops.paged_prefill_attention(out, q, ck, cv, kn, vn, R, table, d, st, page, H, Hkv, bits, ws)
            b.record()
            torch.cuda.synchronize()
            best.append(a.elapsed_time(b))
        return min(best)

    assert us([30000 + chunk] + [900] * 63, [chunk] + [1] * 63) < 4.5 * us([30000 + chunk], [chunk])


def test_a_step_without_tokens():
    # every call of a step takes empty arrays; nothing is launched but the plan
    rng = np.random.default_rng(1)
    G, H, Hkv, page = 3, 16, 8, 32
    table, q, out, ck, cv, kn, vn, R, _ = attention_inputs(rng, [40, 0, 7], H, Hkv, 4, page, T=0)
    q, out = q.contiguous(), out.contiguous()
    lens, start, count, slots = i32([40, 0, 7]), i32([9] * 4), i32([2]), torch.zeros(0, dtype=torch.int64, device="cuda")
    kv = torch.zeros(0, Hkv * 128, dtype=torch.float16, device="cuda")
    before = [x.clone() for x in (ck, kn.view(torch.int16), cv, vn.view(torch.int16))]
    ops.page_plan(table, i32([0, 1, 2, 3]), count, count, lens, i32([0, 0, 0]), None, page, lens, start, slots)
    ops.paged_append(ck, kn, cv, vn, kv, kv, R, slots, Hkv, 4)
    ops.paged_read(kv, kv, ck, kn, cv, vn, R, slots, Hkv, 4)
    ops.paged_prefill_attention(out, q, ck, cv, kn, vn, R, table, lens, start, page, H, Hkv, 4, ops.paged_workspace(0, G, H))
    assert lens.tolist() == [40, 0, 7] and start.tolist() == [0] * 4 and int(count) == 2
    assert all(torch.equal(a, b) for a, b in zip(before, (ck, kn.view(torch.int16), cv, vn.view(torch.int16))))


# ---- offsets of more than 32 bits ---------------------------------------------------------------------------------------------------
def test_pages_behind_the_first_4_gigabytes():
    # the same rows in a small pool and at the end of one whose code arrays pass 4 GB and 2^32 bytes of offsets: the same bytes, rows and results
    rng = np.random.default_rng(21)
    H, Hkv, bits, page, G, R = 32, 8, 4, 64, 4, pu.rotation(6).cuda()
    lens, new = [900, 64, 2500, 31], [40, 5, 600, 1]
    start = [0] + np.cumsum(new).tolist()
    small = 80
    far = (9 << 20) // page  # pages: 9 Mi rows of 512 bytes
    table, used = pu.tables(rng, lens, page)
    assert used <= small
    tables = [table, torch.where(table >= 0, table + (far - small), table)]
    pools = [[torch.empty(n * page, w, dtype=t, device="cuda") for w, t in ((Hkv * 64, torch.uint8), (Hkv, torch.float16)) * 2] for n in (small, far)]
    k, v = (torch.from_numpy(rng.standard_normal((sum(lens), Hkv * 128)).astype(np.float16)).cuda() for _ in range(2))
    q = torch.from_numpy(rng.standard_normal((start[-1], H * 128)).astype(np.float16)).cuda()
    ws, results = ops.paged_workspace(start[-1], G, H), []
    for t, (ck, kn, cv, vn) in zip(tables, pools):
        slots = torch.cat([pu.rows_of(t[g], n, page) for g, n in enumerate(lens)])
        cut = 200  # (a first part by the form for few tokens)
        for a, b in ((0, cut), (cut, sum(lens))):
            ops.paged_append(ck, kn, cv, vn, k[a:b], v[a:b], R, slots[a:b], Hkv, bits)
        k_out, v_out, out, one, wide = torch.empty_like(k), torch.empty_like(v), torch.empty_like(q), torch.empty_like(q[:G]), torch.empty_like(q[:G])
        ops.paged_read(k_out, v_out, ck, kn, cv, vn, R, slots, Hkv, bits)
        ops.paged_prefill_attention(out, q, ck, cv, kn, vn, R, t, i32(lens), i32(start), page, H, Hkv, bits, ws)
        long = torch.empty(1, H * 128, dtype=torch.float16, device="cuda")
        lone = torch.empty_like(q[:20])
        ops.paged_prefill_attention(lone, q[:20], ck, cv, kn, vn, R, t[2:3], i32(lens[2:3]), i32([0, 20]), page, H, Hkv, bits, ws)  # cut along the context
        ops.paged_decode_attention(one, q[:G], ck, cv, kn, vn, R, t, i32(lens), page, H, Hkv, bits, ws)
        ops.paged_decode_attention(long, q[:1], ck, cv, kn, vn, R, t[2:3, :1], i32(lens[2:3]), page, H, Hkv, bits, ws)
        more = torch.cat([t, torch.full((G, 400), -1, dtype=torch.int32, device="cuda")], 1)  # (a bound for which the streaming form is taken)
        ops.paged_decode_attention(wide, q[:G], ck, cv, kn, vn, R, more, i32(lens), page, H, Hkv, bits, ws)
        torch.cuda.synchronize()
        results.append([k_out, v_out, out, lone, one, long, wide, *(x[slots].view(torch.uint8) for x in (ck, kn, cv, vn))])
    for i, (a, b) in enumerate(zip(*results)):
        assert torch.equal(a, b), i
    ck, kn, cv, vn = pools[1]
    for got, at, st in ((results[1][2], lens, start), (results[1][4], lens, list(range(G + 1))), (results[1][6], lens, list(range(G + 1)))):
        pu.assert_attention(got, pu.attention(q[:st[-1]], ck, cv, kn, vn, R, tables[1], at, st, page, H, Hkv, bits))


@pytest.mark.parametrize("T, G", [(340, 34), (40, 40), (330, 2)])
def test_rows_far_apart(T, G):
    # strides that put the last rows more than 2^32 bytes behind the first
    rng = np.random.default_rng(T)
    H, Hkv, bits, page, R = 16, 8, 4, 64, pu.rotation(7).cuda()
    new = [T // G] * G
    lens, start = [n + 50 + 7 * g for g, n in enumerate(new)], [T // G * g for g in range(G + 1)]
    stride = ((5 << 29) // T + 4096) // 8 * 8  # halves: 5 GB of them
    whole = torch.empty(T * stride, dtype=torch.float16, device="cuda")
    column = lambda at, heads: whole.as_strided((T, heads * 128), (stride, 1), at)  # noqa: E731
    table, q, _, ck, cv, kn, vn, _, _ = attention_inputs(rng, lens, H, Hkv, bits, page, T=T)
    kv = torch.from_numpy(rng.standard_normal((T, 2 * Hkv * 128)).astype(np.float16)).cuda()
    far_q, far_k, far_v = column(0, H), column(2048, Hkv), column(2048 + Hkv * 128 + 8, Hkv)
    slots = torch.cat([pu.rows_of(table[g], n, page)[n - new[g]:] for g, n in enumerate(lens)])
    ws = ops.paged_workspace(T, G, H)
    k, v = kv[:, :Hkv * 128], kv[:, Hkv * 128:]
    caches = [[x.clone() for x in (ck, kn, cv, vn)] for _ in range(2)]
    far_k.copy_(k)
    far_v.copy_(v)
    for (c, n, d, m), a, b in zip(caches, (k, far_k), (v, far_v)):
        ops.paged_append(c, n, d, m, a, b, R, slots, Hkv, bits)
    for x, y in zip(*caches):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    c, n, d, m = caches[0]
    near_k, near_v = torch.empty_like(k), torch.empty_like(v)
    ops.paged_read(near_k, near_v, c, n, d, m, R, slots, Hkv, bits)
    ops.paged_read(far_k, far_v, c, n, d, m, R, slots, Hkv, bits)
    assert torch.equal(near_k, far_k) and torch.equal(near_v, far_v)
    far_q.copy_(q)
    near = torch.empty(T, H * 128, dtype=torch.float16, device="cuda")
    calls = [lambda o, a: ops.paged_prefill_attention(o, a, c, d, n, m, R, table, i32(lens), i32(start), page, H, Hkv, bits, ws)]
    if T == G:
        calls.append(lambda o, a: ops.paged_decode_attention(o, a, c, d, n, m, R, table, i32(lens), page, H, Hkv, bits, ws))
    for call in calls:
        call(near, q)
        mid = torch.empty(T, H * 128, dtype=torch.float16, device="cuda")
        call(mid, far_q)                 # queries far apart
        far_res = column(2048, H)        # (where K and V were)
        far_res.fill_(7.0)
        call(far_res, far_q)             # both: columns of one array
        torch.cuda.synchronize()
        assert torch.equal(mid, near) and torch.equal(far_res, near)


# ---- whole steps, two at a time, and captured ---------------------------------------------------------------------------------------
class Loop:
    """A pool, its requests, and three kinds of step: prompts, single tokens beside a chunk, a decode step."""

    def __init__(self, seed, H=32, Hkv=8, bits=4, page=32, G=6, width=80):
        rng = np.random.default_rng(seed)
        self.a, self.page, self.G, self.T = (H, Hkv, bits), page, G, 2600
        pool = G * width // 2
        self.R, self.table = pu.rotation(seed).cuda(), i32(np.full((G, width), -1))
        self.stack, self.count, self.lens = i32(rng.permutation(pool)), i32([pool]), i32(np.zeros(G))
        self.cache = [torch.zeros(pool * page, w, dtype=t, device="cuda") for w, t in ((Hkv * 16 * bits, torch.uint8), (Hkv, torch.float16)) * 2]
        self.start, self.slots, self.pos = i32(np.zeros(G + 1)), torch.zeros(self.T, dtype=torch.int64, device="cuda"), i32(np.zeros(self.T))
        self.ws = ops.paged_workspace(self.T, G, H)
        self.steps = [rng.integers(100, 400, G), np.where(np.arange(G) == 2, 150, 1), np.ones(G, int), np.where(np.arange(G) == 4, 0, 1)]
        self.ended = [None, None, np.arange(G) % 3 == 0, None]
        self.steps[2] = np.where(np.arange(G) % 3 == 0, 37, 1)
        self.steps = [i32(s) for s in self.steps]
        self.ended = [None if e is None else torch.from_numpy(e).cuda() for e in self.ended]
        self.qkv = [torch.from_numpy(rng.standard_normal((self.T, (H + 2 * Hkv) * 128)).astype(np.float16)).cuda() for _ in range(4)]
        self.out = [torch.zeros(self.T, H * 128, dtype=torch.float16, device="cuda") for _ in range(5)]

    def run(self):
        (H, Hkv, bits), (ck, kn, cv, vn) = self.a, self.cache
        for i in range(4):
            q, k, v = self.qkv[i][:, :H * 128], self.qkv[i][:, H * 128:(H + Hkv) * 128], self.qkv[i][:, (H + Hkv) * 128:]
            ops.page_plan(self.table, self.stack, self.count, self.count, self.lens, self.steps[i], self.ended[i], self.page, self.lens, self.start, self.slots, self.pos)
            ops.paged_append(ck, kn, cv, vn, k, v, self.R, self.slots, Hkv, bits)
            ops.paged_prefill_attention(self.out[i], q, ck, cv, kn, vn, self.R, self.table, self.lens, self.start, self.page, H, Hkv, bits, self.ws)
        ops.paged_decode_attention(self.out[4][:self.G], self.qkv[3][:self.G, :H * 128], ck, cv, kn, vn, self.R, self.table, self.lens, self.page, H, Hkv, bits, self.ws)

    def state(self):
        return [self.table, self.stack, self.count, self.lens, self.start, self.slots, self.pos, *(x.view(torch.uint8) for x in self.cache), *self.out]


def test_steps_on_two_streams_and_from_one_graph():
    want = []
    for seed in (1, 2):
        loop = Loop(seed)
        loop.run()
        torch.cuda.synchronize()
        assert loop.lens.min() > 0 and int(loop.count) >= 0
        want.append([x.clone() for x in loop.state()])
    for _ in range(4):
        loops, streams = [Loop(1), Loop(2)], [torch.cuda.Stream() for _ in range(2)]
        torch.cuda.synchronize()
        for loop, s in zip(loops, streams):
            with torch.cuda.stream(s):
                loop.run()
        torch.cuda.synchronize()
        for loop, w in zip(loops, want):
            assert all(torch.equal(a, b) for a, b in zip(loop.state(), w))
    loop, graph = Loop(1), torch.cuda.CUDAGraph()
    keep = [x.clone() for x in loop.state()]
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        loop.run()
    for _ in range(3):
        for a, b in zip(loop.state(), keep):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(loop.state(), want[0]))
