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
