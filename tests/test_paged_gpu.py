"""Paged caches on the GPU: plans against whole numbers, appends against the launchers' bytes, reads and attention against 64 bits."""
import pathlib
import subprocess
import sys

import numpy as np
import pytest
import torch

from tests import paged_util as pu

pytestmark = pytest.mark.gpu
gu = pytest.importorskip("tests.gpu_util")
from triebwerk_b200 import TqError, ops  # noqa: E402


def i32(a):
    return torch.as_tensor(np.ascontiguousarray(a), dtype=torch.int32).cuda()


@pytest.fixture(autouse=True)
def no_status():
    yield
    assert ops.paged_status() == 0


# ---- plan -----------------------------------------------------------------------------------------------------------------
def plan_case(rng, G, page, width, most_new, spare, ended=0.0, one=False):
    context = rng.integers(0, width * page // 2 + 1, G)
    new = np.ones(G, np.int64) if one else rng.integers(0, most_new + 1, G)
    finished = (rng.random(G) < ended).astype(np.uint8)
    need = -(-context // page)
    pool = int(need.sum()) + spare
    order = rng.permutation(pool)
    table = np.full((G, width), -3, np.int64)
    at = 0
    for g, n in enumerate(need):
        table[g, :n] = order[at:at + n]
        at += n
    stack = np.full(pool, -9, np.int64)
    stack[:pool - at] = order[at:]
    return table, stack, pool - at, context, new, finished


def run_plan(table, stack, count, context, new, finished, page, T, wide=0, positions=True, in_place=False):
    G, width = table.shape
    store = i32(np.concatenate([table, np.full((G, wide), 77)], 1))
    d = dict(stack=i32(stack), count=i32([count]), context=i32(context), new=i32(new), fin=None if finished is None else torch.from_numpy(finished).cuda())
    lens = d["context"] if in_place else torch.full((G,), 99, dtype=torch.int32, device="cuda")
    out = d["count"] if in_place else torch.full((1,), 99, dtype=torch.int32, device="cuda")
    start = torch.full((G + 1,), 99, dtype=torch.int32, device="cuda")
    slots = torch.full((T,), 99, dtype=torch.int64, device="cuda")
    pos = torch.full((T,), 99, dtype=torch.int32, device="cuda") if positions else None
    ops.page_plan(store[:, :width], d["stack"], d["count"], out, d["context"], d["new"], d["fin"], page, lens, start, slots, pos)
    torch.cuda.synchronize()
    assert (store[:, width:] == 77).all()
    return [x.cpu().numpy().tolist() if x is not None else None for x in (lens, start, slots, pos, out, store[:, :width], d["stack"])]


def check_plan(table, stack, count, context, new, finished, page, T, **kw):
    got = run_plan(table, stack, count, context, new, finished, page, T, **kw)
    t, st = table.copy(), stack.copy()
    want = pu.plan(t, st, count, [int(c) for c in context], new, finished, page, T)
    for name, a, b in zip(("lens", "start", "slots", "positions"), got, want):
        assert a is None or a == list(b), name
    assert got[4] == [want[4]]
    assert got[5] == t.tolist()
    assert got[6] == st.tolist()
    return want


@pytest.mark.parametrize("G", [1, 2, 31, 33, 256, 1023, 1025, 2500])
@pytest.mark.parametrize("page", [32, 64, 1024])
def test_plan_decode_step(G, page):
    rng = np.random.default_rng(G + page)
    check_plan(*plan_case(rng, G, page, 5, 1, G + 7, ended=0.1, one=True), page, G, wide=3)


@pytest.mark.parametrize("G, most_new, T", [(1, 1, 1), (1, 700, 900), (7, 300, 2100), (40, 90, 3600), (3, 4000, 12500), (64, 500, 32003), (1300, 40, 60000),
                                            (9000, 3, 30000)])
def test_plan_prompts(G, most_new, T):
    rng = np.random.default_rng(G)
    width = 2 * (most_new // 32 + 2)
    check_plan(*plan_case(rng, G, 32, width, most_new, G * (most_new // 32 + 2), ended=0.2), 32, T)


@pytest.mark.parametrize("T", [0, 100, 3000, 9000])
def test_plan_runs_out(T):
    # too few pages, too short a slot map, requests that fit no row
    rng = np.random.default_rng(T)
    table, stack, count, context, new, finished = plan_case(rng, 60, 32, 12, 200, 90, ended=0.1)
    context[5] = 12 * 32 - 1
    table[5] = rng.permutation(12)
    new[5], new[9], new[11] = 2, -4, 0
    want = check_plan(table, stack, count, context, new, finished, 32, T)
    assert any(n < 0 for n in want[0]) and any(n > 0 for n in want[0])


def test_plan_ended_row_is_taken_again_and_in_place():
    rng = np.random.default_rng(3)
    table, stack, count, context, new, finished = plan_case(rng, 50, 64, 9, 200, 12, ended=0.5)
    context = np.where(rng.random(50) < 0.3, ~context, context)  # (not admitted in the step before)
    new[finished != 0] = 130
    check_plan(table, stack, count, context, new, finished, 64, 9000, in_place=True)
    check_plan(table, stack, count, context, new, None, 64, 4000, positions=False)
    finished = finished.astype(bool)
    check_plan(table, stack, count, context, new, finished, 64, 4096)


def test_plan_strange_counts():
    rng = np.random.default_rng(4)
    table, stack, count, context, new, finished = plan_case(rng, 6, 32, 4, 40, 20)
    check_plan(table, stack, -5, context, new, finished, 32, 300)
    stack[:] = np.arange(len(stack))
    check_plan(table, stack, len(stack) + 100, context, new, np.ones(6, np.uint8), 32, 300)  # (a full stack takes no more)
    check_plan(table, stack, 10, np.full(6, 2**31 - 1), new, finished, 32, 300)               # (lengths beyond every row)


def test_plan_captured_steps():
    # a loop of decode steps in place, replayed from one graph
    rng = np.random.default_rng(5)
    G, page, width = 37, 32, 6
    table, stack, count, context, _, _ = plan_case(rng, G, page, width, 1, 60)
    new = np.ones(G, np.int64)
    d = [i32(x) for x in (table, stack, [count], context, new)]
    start, slots, pos = torch.zeros(G + 1, dtype=torch.int32, device="cuda"), torch.zeros(G, dtype=torch.int64, device="cuda"), i32(np.zeros(G))
    call = lambda: ops.page_plan(d[0], d[1], d[2], d[2], d[3], d[4], None, page, d[3], start, slots, pos)  # noqa: E731
    keep = [x.clone() for x in d]
    call()
    for x, k in zip(d, keep):
        x.copy_(k)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    t, st, c, ctx = table.copy(), stack.copy(), count, [int(x) for x in context]
    for _ in range(40):
        graph.replay()
        ctx, _, want, _, c = pu.plan(t, st, c, ctx, new, None, page, G)
        assert slots.tolist() == want
    assert d[3].tolist() == ctx and d[2].tolist() == [c] and d[0].tolist() == t.tolist()


# ---- append and read --------------------------------------------------------------------------------------------------------
def store_inputs(rng, T, Hkv, bits, page=32, fused=True, pad=True):
    rows = (T // page + 3) * page * 2
    slots = rng.permutation(rows)[:T].astype(np.int64)
    if pad and T > 3:
        slots[rng.integers(0, T, T // 16 + 1)] = -1
        slots[1] = rows          # just outside
        slots[2] = 1 << 40
    kv = rng.standard_normal((T, 3 * Hkv * 128)).astype(np.float16)
    kv[0, :] = 0                 # all zero
    if T > 5:
        kv[5, :200] *= np.float16(1000.0)
    kv = torch.from_numpy(kv).cuda()
    k, v = kv[:, Hkv * 128:2 * Hkv * 128], kv[:, 2 * Hkv * 128:]
    if not fused:
        k, v = k.contiguous(), v.contiguous()
    caches = [pu.random_cache(rng, rows, Hkv, bits) for _ in range(2)]
    return rows, torch.from_numpy(slots).cuda(), k, v, caches


@pytest.mark.parametrize("bits", [4, 2])
@pytest.mark.parametrize("Hkv", [8, 4, 3, 1, 16])
@pytest.mark.parametrize("T", [1, 2, 17, 64, 591, 593, 1500])
def test_append_stores_the_launchers_bytes(T, Hkv, bits):
    rng = np.random.default_rng(T * 100 + Hkv + bits)
    rows, slots, k, v, ((ck, kn), (cv, vn)) = store_inputs(rng, T, Hkv, bits, fused=T % 2 == 0)
    R = pu.rotation(1).cuda()
    before = [x.clone() for x in (ck, kn, cv, vn)]
    ops.paged_append(ck, kn, cv, vn, k, v, R, slots, Hkv, bits)
    torch.cuda.synchronize()
    keep = (slots >= 0) & (slots < rows)
    for x, codes, norms, old_codes, old_norms in ((k, ck, kn, before[0], before[1]), (v, cv, vn, before[2], before[3])):
        pos = slots[keep].to(torch.int32)
        if pos.numel():
            from triebwerk_b200 import ops as o
            o.launch_turbo_kv_quantize(old_codes, old_norms, x[keep].contiguous(), R, pos, rows, int(pos.numel()), Hkv, 128, Hkv * 128, bits)
        assert torch.equal(codes, old_codes)
        assert torch.equal(norms.view(torch.int16), old_norms.view(torch.int16))


@pytest.mark.parametrize("bits", [4, 2])
@pytest.mark.parametrize("Hkv", [8, 5, 1])
@pytest.mark.parametrize("T", [1, 3, 64, 1111])
def test_read_gives_what_rows_stand_for(T, Hkv, bits):
    rng = np.random.default_rng(T + Hkv + bits)
    rows, slots, _, _, ((ck, kn), (cv, vn)) = store_inputs(rng, T, Hkv, bits)
    kn[rows // 2, 0] = float("nan")  # (a norm that only its own row's vector takes)
    R = pu.rotation(2).cuda()
    wide = torch.full((T, 2 * Hkv * 128 + 16), 5.0, dtype=torch.float16, device="cuda")
    k_out, v_out = wide[:, :Hkv * 128], wide[:, Hkv * 128 + 8:2 * Hkv * 128 + 8]
    ops.paged_read(k_out, v_out, ck, kn, cv, vn, R, slots, Hkv, bits)
    torch.cuda.synchronize()
    keep = (slots >= 0) & (slots < rows)
    at = torch.where(keep, slots, 0)
    for got, codes, norms in ((k_out, ck, kn), (v_out, cv, vn)):
        want = torch.where(keep[:, None], pu.vectors(codes[at], norms[at], R, bits).reshape(T, -1), 0.0)
        bad = want.isnan()
        assert torch.equal(got.isnan(), bad)
        # centroids rounded to fp16 (2^-11 each, in a sum of 128 products with |c| |R| of 2-norm norm * 1), the result rounded once (2^-11)
        tol = 2.0**-11 * want.abs() + 2.0**-11 * torch.where(keep[:, None], norms[at].double().repeat_interleave(128, 1), 0.0)
        assert ((got.double() - want).abs()[~bad] <= tol[~bad]).all()
    assert (wide[:, Hkv * 128:Hkv * 128 + 8] == 5).all() and (wide[:, 2 * Hkv * 128 + 8:] == 5).all()


# ---- decode attention ---------------------------------------------------------------------------------------------------------
def attention_inputs(rng, lens, H, Hkv, bits, page, T=None, extra_columns=1, strided=True):
    table, pool = pu.tables(rng, lens, page, extra_columns=extra_columns)
    rows = pool * page
    (ck, kn), (cv, vn) = (pu.random_cache(rng, rows, Hkv, bits) for _ in range(2))
    # what no request holds must not matter: norms that are not numbers in every such row
    held = torch.zeros(rows, dtype=torch.bool, device="cuda")
    for g, n in enumerate(lens):
        if n > 0:
            held[pu.rows_of(table[g], n, page)] = True
    kn[~held], vn[~held] = float("nan"), float("inf")
    T = len(lens) if T is None else T
    qkv = torch.from_numpy(rng.standard_normal((T, H * 128 + 64)).astype(np.float16)).cuda()
    q = qkv[:, :H * 128] if strided else qkv[:, :H * 128].contiguous()
    out = torch.full((T, H * 128 + 8), 7.0, dtype=torch.float16, device="cuda")
    return table, q, out[:, :H * 128], ck, cv, kn, vn, pu.rotation(3).cuda(), out


def check_decode(lens, H, Hkv, bits, page, seed, narrow=False, strided=True):
    rng = np.random.default_rng(seed)
    table, q, out, ck, cv, kn, vn, R, whole = attention_inputs(rng, lens, H, Hkv, bits, page, extra_columns=0 if narrow else 1, strided=strided)
    ws = ops.paged_workspace(len(lens), len(lens), H)
    ops.paged_decode_attention(out, q, ck, cv, kn, vn, R, table, i32(lens), page, H, Hkv, bits, ws)
    torch.cuda.synchronize()
    most = table.shape[1] * page
    cut = [min(n, most) for n in lens]
    want = pu.attention(q, ck, cv, kn, vn, R, table, cut, list(range(len(lens) + 1)), page, H, Hkv, bits)
    pu.assert_attention(out, want, f"{bits}-bit {H}/{Hkv} page {page}")
    for g, n in enumerate(lens):
        assert n > 0 or (out[g] == 0).all()
    assert (whole[:, H * 128:] == 7).all()


@pytest.mark.parametrize("bits", [4, 2])
@pytest.mark.parametrize("H, Hkv", [(16, 8), (32, 8), (32, 4), (4, 4), (40, 8), (14, 2), (9, 3), (16, 1)])
@pytest.mark.parametrize("page", [32, 128])
def test_decode_small_batches(H, Hkv, bits, page):
    check_decode([0, 1, 31, 32, 33, 64, 65, 0, 500], H, Hkv, bits, page, H + Hkv + bits + page)
    check_decode([777], H, Hkv, bits, page, 1)


@pytest.mark.parametrize("bits", [4, 2])
@pytest.mark.parametrize("H, Hkv", [(16, 8), (32, 8), (32, 4), (16, 4)])
@pytest.mark.parametrize("page", [32, 64, 256])
def test_decode_streaming_form(H, Hkv, bits, page):
    # batches of many tokens: the streaming kernels, empty places at both ends and in a row
    rng = np.random.default_rng(page)
    lens = [0, 0] + rng.integers(1, 3000, 60).tolist() + [0, 0, 0] + rng.integers(1, 4500, 40).tolist() + [1, 32, 33, 0]
    check_decode(lens, H, Hkv, bits, page, H + Hkv + bits + page)
    check_decode([9000, 0, 16000, 1], H, Hkv, bits, page, 2, strided=False)


@pytest.mark.parametrize("bits", [4, 2])
def test_decode_no_tokens_at_all(bits):
    for lens in ([0], [0] * 200, [-1, -500, 0] * 40):
        check_decode(lens, 16, 8, bits, 64, 5)


def empty_wide(G, H, Hkv, bits):
    """A batch without tokens whose table has room for many: the streaming form by its bound."""
    table = torch.zeros(G, 200, dtype=torch.int32, device="cuda")
    rng = np.random.default_rng(0)
    (ck, kn), (cv, vn) = (pu.random_cache(rng, 64 * 4, Hkv, bits) for _ in range(2))
    q = torch.ones(G, H * 128, dtype=torch.float16, device="cuda")
    out = torch.full_like(q, 3.0)
    return out, q, ck, cv, kn, vn, pu.rotation(0).cuda(), table


@pytest.mark.parametrize("H, Hkv, bits", [(16, 8, 4), (32, 8, 2), (32, 4, 4)])
def test_decode_no_tokens_in_wide_tables(H, Hkv, bits):
    args = empty_wide(64, H, Hkv, bits)
    lens = i32(np.zeros(64))
    ws = ops.paged_workspace(64, 64, H)
    for _ in range(3):
        ops.paged_decode_attention(*args, lens, 64, H, Hkv, bits, ws)
    assert (args[0] == 0).all()
    lens[40] = 1
    ops.paged_decode_attention(*args, lens, 64, H, Hkv, bits, ws)
    assert (args[0][40] != 0).any() and (args[0][:40] == 0).all() and (args[0][41:] == 0).all()


def test_decode_many_requests():
    rng = np.random.default_rng(7)
    check_decode(rng.integers(0, 90, 1023).tolist(), 16, 8, 4, 32, 8)
    check_decode(rng.integers(0, 90, 1400).tolist(), 16, 8, 4, 32, 9)


def test_decode_lengths_beyond_the_table_are_cut():
    rng = np.random.default_rng(11)
    lens = [64, 128, 96]
    table, q, out, ck, cv, kn, vn, R, _ = attention_inputs(rng, lens, 16, 8, 4, 32, extra_columns=0)
    ws = ops.paged_workspace(3, 3, 16)
    ops.paged_decode_attention(out, q, ck, cv, kn, vn, R, table, i32([64, 1 << 30, 96]), 32, 16, 8, 4, ws)
    want = pu.attention(q, ck, cv, kn, vn, R, table, lens, [0, 1, 2, 3], 32, 16, 8, 4)
    pu.assert_attention(out, want)


@pytest.mark.parametrize("H, Hkv, G, n", [(16, 8, 4, 600), (16, 8, 64, 3000)])
def test_decode_shared_pages_narrow_views_and_streams(H, Hkv, G, n):
    # rollouts whose rows name the same prompt pages; a view of a wider table; another stream, captured and replayed with new lengths
    rng = np.random.default_rng(12)
    lens = [n] * G
    table, q, out, ck, cv, kn, vn, R, _ = attention_inputs(rng, lens, H, Hkv, 4, 64)
    table[1:, :n // 128] = table[0, :n // 128]
    wide = torch.cat([table, torch.full((G, 50), -1, dtype=torch.int32, device="cuda")], 1)
    view, d = wide[:, :table.shape[1]], i32(lens)
    ws = ops.paged_workspace(G, G, H)
    call = lambda: ops.paged_decode_attention(out, q, ck, cv, kn, vn, R, view, d, 64, H, Hkv, 4, ws)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    side.synchronize()
    check = lambda cut: pu.assert_attention(out, pu.attention(q, ck, cv, kn, vn, R, table, cut, list(range(G + 1)), 64, H, Hkv, 4))  # noqa: E731
    check(lens)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for cut in ([n // 2] * G, [0] * G, [(37 * g) % n for g in range(G)]):
        d.copy_(i32(cut))
        out.fill_(9.0)
        graph.replay()
        torch.cuda.synchronize()
        check(cut)


def test_decode_infinite_and_missing_norms():
    # a norm that is not a number poisons its own request and no other
    rng = np.random.default_rng(13)
    lens = [40, 700, 40]
    table, q, out, ck, cv, kn, vn, R, _ = attention_inputs(rng, lens, 16, 8, 4, 32)
    ws = ops.paged_workspace(3, 3, 16)
    vn[pu.rows_of(table[1], 700, 32)[333]] = float("nan")
    ops.paged_decode_attention(out, q, ck, cv, kn, vn, R, table, i32(lens), 32, 16, 8, 4, ws)
    assert out[1].isnan().all() and out[0].isfinite().all() and out[2].isfinite().all()


def test_python_refusals():
    rng = np.random.default_rng(14)
    table, q, out, ck, cv, kn, vn, R, _ = attention_inputs(rng, [40, 50], 16, 8, 4, 32)
    lens, ws = i32([40, 50]), ops.paged_workspace(2, 2, 16)
    good = [out, q, ck, cv, kn, vn, R, table, lens, 32, 16, 8, 4, ws]
    for at, bad in ((0, out.float()), (1, q[:1]), (1, q[:, ::2]), (2, ck.cpu()), (2, ck[:-1]), (3, cv[:32]), (4, kn.float()), (6, R[:64]), (7, table.long()),
                    (7, table.t()), (8, lens.long()), (8, lens[:1]), (9, 48), (10, 15), (11, 4), (12, 3), (13, ws.float()), (0, None), (10, "x")):
        args = list(good)
        args[at] = bad
        with pytest.raises((AssertionError, TqError)):
            ops.paged_decode_attention(*args)
    with pytest.raises(TqError):
        ops.paged_decode_attention(*good[:13], ws[:1024])
    with pytest.raises(TypeError):
        ops.paged_decode_attention(*good, 1) if False else ops.hostcall.paged_decode_attention(*good, 1)
    k = torch.zeros(2, 1024, dtype=torch.float16, device="cuda")
    slots = torch.zeros(2, dtype=torch.int64, device="cuda")
    for bad in ((k, k[:1], slots), (k, k.float(), slots), (k, k, slots.int()), (k, k, slots[:1]), (k, k.cpu(), slots), (k[:, :512], k[:, :512], slots)):
        with pytest.raises((AssertionError, TqError)):
            ops.paged_append(ck, kn, cv, vn, bad[0], bad[1], R, bad[2], 8, 4)


# ---- prefill attention ----------------------------------------------------------------------------------------------------------
def check_prefill(lens, new, H, Hkv, bits, page, seed, tail=3, narrow=False, strided=True):
    rng = np.random.default_rng(seed)
    start = [0] + np.cumsum(new).tolist()
    T = start[-1] + tail
    table, q, out, ck, cv, kn, vn, R, whole = attention_inputs(rng, lens, H, Hkv, bits, page, T=T, extra_columns=0 if narrow else 1, strided=strided)
    ws = ops.paged_workspace(T, len(lens), H)
    ops.paged_prefill_attention(out, q, ck, cv, kn, vn, R, table, i32(lens), i32(start), page, H, Hkv, bits, ws)
    torch.cuda.synchronize()
    want = pu.attention(q, ck, cv, kn, vn, R, table, lens, start, page, H, Hkv, bits)
    pu.assert_attention(out[:start[-1]], (want[0][:start[-1]], want[1][:start[-1]]), f"{bits}-bit {H}/{Hkv} page {page}")
    for g, n in enumerate(lens):  # queries with nothing in front of them
        none = out[start[g]:start[g + 1]][:max(0, new[g] - max(n, 0))]
        assert (none == 0).all()
    assert (whole[:, H * 128:] == 7).all() and (whole[start[-1]:] == 7).all()


@pytest.mark.parametrize("bits", [4, 2])
@pytest.mark.parametrize("H, Hkv", [(16, 8), (32, 8), (4, 4), (40, 8), (14, 2), (16, 1), (9, 3)])
@pytest.mark.parametrize("page", [32, 128])
def test_prefill_small_batches(H, Hkv, bits, page):
    new = [1, 0, 5, 33, 128, 1, 70, 0, 64]
    lens = [1, 0, 5, 40, 128, 300, 71, 90, 1000]
    check_prefill(lens, new, H, Hkv, bits, page, H + Hkv + bits + page)
    check_prefill([77], [77], H, Hkv, bits, page, 1, tail=0)


@pytest.mark.parametrize("bits", [4, 2])
@pytest.mark.parametrize("H, Hkv", [(16, 8), (32, 8), (32, 4), (40, 8)])
@pytest.mark.parametrize("page", [32, 64, 256])
def test_prefill_two_blocks_a_cta(H, Hkv, bits, page):
    rng = np.random.default_rng(page)
    new = rng.integers(1, 700, 14).tolist() + [0, 1, 129, 512, 127]
    lens = [n + c for n, c in zip(new, [0, 0, 1000, 31, 32, 33, 500, 1, 0, 7, 128, 127, 129, 900, 64, 2000, 0, 0, 1])]
    check_prefill(lens, new, H, Hkv, bits, page, H + Hkv + bits + page)


@pytest.mark.parametrize("bits", [4, 2])
@pytest.mark.parametrize("H, Hkv, new, lens", [(16, 8, [4], [9000]), (32, 8, [1, 5], [5000, 700]), (16, 1, [8, 1, 3], [4000, 1, 3]), (14, 2, [40], [6000]),
                                               (8, 1, [17], [16001])])
def test_prefill_cut_along_the_context(H, Hkv, new, lens, bits):
    check_prefill(lens, new, H, Hkv, bits, 64, sum(lens), tail=2)


@pytest.mark.parametrize("bits", [4, 2])
def test_prefill_rows_without_tokens(bits):
    # requests not admitted, empty ones, more queries than tokens: zeros
    check_prefill([-5, 0, 3, 200, -1, 10], [7, 2, 8, 200, 1, 140], 16, 8, bits, 32, 3)
    check_prefill([0], [300], 16, 8, bits, 32, 4)
    check_prefill([-9] * 40, [130] * 40, 16, 8, bits, 32, 5)
    check_prefill([0, 5000], [3, 3], 16, 1, bits, 32, 6)


def test_prefill_many_requests():
    rng = np.random.default_rng(8)
    new = rng.integers(0, 4, 900)
    check_prefill((new + rng.integers(0, 60, 900)).tolist(), new.tolist(), 16, 8, 4, 32, 9)


def test_prefill_single_tokens_are_a_decode_step():
    rng = np.random.default_rng(10)
    lens = rng.integers(1, 900, 20).tolist()
    check_prefill(lens, [1] * 20, 32, 8, 4, 32, 11, tail=0)


@pytest.mark.parametrize("H, Hkv, n, L", [(16, 8, 40, 900), (16, 1, 4, 5000), (16, 8, 600, 600)])
def test_prefill_captured_on_another_stream(H, Hkv, n, L):
    rng = np.random.default_rng(12)
    G = 6
    lens, start = [L] * G, [n * g for g in range(G + 1)]
    table, q, out, ck, cv, kn, vn, R, _ = attention_inputs(rng, lens, H, Hkv, 4, 64, T=n * G)
    d, st = i32(lens), i32(start)
    ws = ops.paged_workspace(n * G, G, H)
    call = lambda: ops.paged_prefill_attention(out, q, ck, cv, kn, vn, R, table, d, st, 64, H, Hkv, 4, ws)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for cut in (lens, [n] * G, [0] * G, [L - 13 * g for g in range(G)]):
        d.copy_(i32(cut))
        out.fill_(9.0)
        graph.replay()
        torch.cuda.synchronize()
        pu.assert_attention(out, pu.attention(q, ck, cv, kn, vn, R, table, cut, start, 64, H, Hkv, 4))


def test_prefill_norms_that_are_not_finite():
    # of a later token: nothing of it reaches the earlier ones; of an earlier token: every query behind it
    rng = np.random.default_rng(13)
    lens, new, start = [300, 300], [300, 300], [0, 300, 600]
    for name, value in (("v", float("nan")), ("v", float("inf")), ("k", float("nan"))):
        table, q, out, ck, cv, kn, vn, R, _ = attention_inputs(rng, lens, 16, 8, 4, 32, T=600)
        at = pu.rows_of(table[0], 300, 32)[150]
        (vn if name == "v" else kn)[at, 3] = value
        ws = ops.paged_workspace(600, 2, 16)
        ops.paged_prefill_attention(out, q, ck, cv, kn, vn, R, table, i32(lens), i32(start), 32, 16, 8, 4, ws)
        bad = ~out.isfinite().view(600, 8, 256).all(-1)
        want = torch.zeros_like(bad)
        want[150:300, 3] = True
        assert torch.equal(bad, want)


@pytest.mark.parametrize("bits", [4, 2])
@pytest.mark.parametrize("H, Hkv, n", [(32, 8, 5), (16, 8, 12), (14, 2, 3), (32, 4, 3), (32, 8, 8), (16, 8, 16), (40, 8, 4), (16, 1, 2)])
@pytest.mark.parametrize("G", [1, 7, 48])
def test_prefill_a_few_tokens_each(H, Hkv, n, G, bits):
    # as in checking drafted tokens: 17 to 24 score rows per KV head, and 32, of every request
    past = [0, 1, 11, 12, 16, 31, 32, 33, 200, 640, 1500, 2111]
    check_prefill([n + past[(5 * g + G) % 12] for g in range(G)], [n] * G, H, Hkv, bits, 32, n + G, tail=0)


def test_prefill_one_prompt_beside_single_tokens():
    rng = np.random.default_rng(17)
    lens = rng.integers(1, 1200, 61).tolist()
    lens[30] = 1500
    check_prefill(lens, [600 if g == 30 else 1 for g in range(61)], 32, 8, 4, 64, 18)


@pytest.mark.parametrize("new, n", [(40, 900), (5, 700)])
def test_prefill_shared_pages_and_two_streams_at_once(new, n):
    # requests whose rows name the same prompt pages; two calls on two streams, each with a workspace of its own
    rng = np.random.default_rng(19)
    G, H, Hkv = 6, 16, 8
    lens, start = [n] * G, [new * g for g in range(G + 1)]
    table, q, out, ck, cv, kn, vn, R, _ = attention_inputs(rng, lens, H, Hkv, 4, 64, T=new * G)
    table[1:, :n // 128] = table[0, :n // 128]
    d, st = i32(lens), i32(start)
    q2, out2 = q.flip(0).contiguous(), torch.empty(new * G, H * 128, dtype=torch.float16, device="cuda")
    work = [ops.paged_workspace(new * G, G, H) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        for s, ws, a, o in zip(streams, work, (q, q2), (out, out2)):
            with torch.cuda.stream(s):
                ops.paged_prefill_attention(o, a, ck, cv, kn, vn, R, table, d, st, 64, H, Hkv, 4, ws)
    torch.cuda.synchronize()
    for a, o in ((q, out), (q2, out2)):
        pu.assert_attention(o, pu.attention(a, ck, cv, kn, vn, R, table, lens, start, 64, H, Hkv, 4))


FIRST_CALLS_CAPTURED = """
import torch
from triebwerk_b200 import ops
R = ops.rotation_matrix().cuda()
ck, cv = (torch.zeros(256, 8 * 64, dtype=torch.uint8, device="cuda") for _ in range(2))
kn, vn = (torch.zeros(256, 8, dtype=torch.float16, device="cuda") for _ in range(2))
k, v, q = (torch.randn(8, n * 128, device="cuda").half() for n in (8, 8, 16))
out, prompt, k2, v2 = (torch.zeros_like(x) for x in (q, q, k, v))
i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
table, stack, count, lens, new, start = torch.zeros(8, 2, dtype=torch.int32, device="cuda"), i32(*range(8)), i32(8), i32(*[0] * 8), i32(*[1] * 8), i32(*[0] * 9)
slots, ws = torch.zeros(8, dtype=torch.int64, device="cuda"), ops.paged_workspace(8, 8, 16)
graph = torch.cuda.CUDAGraph()
torch.cuda.synchronize()
with torch.cuda.graph(graph):
    ops.page_plan(table, stack, count, count, lens, new, None, 32, lens, start, slots)
    ops.paged_append(ck, kn, cv, vn, k, v, R, slots, 8, 4)
    ops.paged_decode_attention(out, q, ck, cv, kn, vn, R, table, lens, 32, 16, 8, 4, ws)
    ops.paged_prefill_attention(prompt, q, ck, cv, kn, vn, R, table, lens, start, 32, 16, 8, 4, ws)
    ops.paged_read(k2, v2, ck, kn, cv, vn, R, slots, 8, 4)
graph.replay()
torch.cuda.synchronize()
assert lens.tolist() == [1] * 8 and int(count) == 0 and ops.paged_status() == 0
# one token each: the attentions give its value back, to five roundings of 2^-11 (weight, centroid, result before and behind R; what was read)
want = v2.view(8, 8, 1, 128).expand(8, 8, 2, 128).reshape(8, -1).double()
for got in (out, prompt):
    assert (got - want).norm() < 5 * 2.0**-11 * want.norm()
assert (v2 - v).double().square().sum() < 0.012 * v.double().square().sum()  # (0.0095: the 4-bit code book's error)
"""


def test_the_first_calls_of_a_process_captured():
    root = str(pathlib.Path(__file__).resolve().parent.parent)
    done = subprocess.run([sys.executable, "-c", FIRST_CALLS_CAPTURED], cwd=root, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


# ---- all together -----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("bits, H, Hkv, page", [(4, 16, 8, 32), (2, 32, 8, 64), (4, 14, 2, 128)])
def test_a_serving_loop(bits, H, Hkv, page):
    """Requests come and go over ten steps: plan, append, attention of prompts and of single tokens, against vectors kept in 64 bits
    (read back from the cache, whose rows are those of the plan)."""
    rng = np.random.default_rng(bits + H)
    G, width, pool = 5, 1024 // page, 4 * 1024 // page
    R = pu.rotation(4).cuda()
    (ck, kn), (cv, vn) = (pu.random_cache(rng, pool * page, Hkv, bits) for _ in range(2))
    table = i32(np.full((G, width), -1))
    stack, count = i32(rng.permutation(pool)), i32([pool])
    lens = i32(np.zeros(G))
    history = [[] for _ in range(G)]  # rows, in order, that each request's tokens went to
    for step in range(10):
        ended = np.array([len(h) > 0 and rng.random() < 0.25 for h in history], np.uint8)
        for g in range(G):
            if ended[g]:
                history[g] = []
        new = np.array([1 if h else int(rng.integers(0, 400)) for h in history])
        if step % 3 == 1:
            new = np.where(new == 1, rng.integers(0, 6, G), new)
        T = int(new.sum()) + 2
        start, slots, pos = i32(np.zeros(G + 1)), torch.zeros(T, dtype=torch.int64, device="cuda"), i32(np.zeros(T))
        ops.page_plan(table, stack, count, count, lens, i32(new), torch.from_numpy(ended).cuda(), page, lens, start, slots, pos)
        qkv = torch.from_numpy(rng.standard_normal((T, (H + 2 * Hkv) * 128)).astype(np.float16)).cuda()
        q, k, v = qkv[:, :H * 128], qkv[:, H * 128:(H + Hkv) * 128], qkv[:, (H + Hkv) * 128:]
        ops.paged_append(ck, kn, cv, vn, k, v, R, slots, Hkv, bits)
        k_back, v_back = torch.empty(T, Hkv * 128, dtype=torch.float16, device="cuda"), torch.empty(T, Hkv * 128, dtype=torch.float16, device="cuda")
        ops.paged_read(k_back, v_back, ck, kn, cv, vn, R, slots, Hkv, bits)
        out = torch.full((T, H * 128), 7.0, dtype=torch.float16, device="cuda")
        ws = ops.paged_workspace(T, G, H)
        ops.paged_prefill_attention(out, q, ck, cv, kn, vn, R, table, lens, start, page, H, Hkv, bits, ws)
        torch.cuda.synchronize()
        at = 0
        for g in range(G):
            for t in range(new[g]):
                assert pos[at] == len(history[g])
                history[g].append(int(slots[at]))
                at += 1
        held = [len(h) for h in history]
        assert lens.tolist() == held and (slots[at:] == -1).all()
        rows = sum(history, [])
        assert len(set(rows)) == len(rows) and int(count) == pool - sum(-(-n // page) for n in held)
        # quantising keeps most of a vector: the error of the 4-bit code book is 0.0095 of the energy, of the 2-bit one 0.1175
        if at:
            for a, b in ((k, k_back), (v, v_back)):
                off = (a[:at].double() - b[:at].double()).square().sum() / a[:at].double().square().sum()
                assert off < {4: 0.012, 2: 0.13}[bits]
        want = pu.attention(q, ck, cv, kn, vn, R, table, held, start.tolist(), page, H, Hkv, bits)
        pu.assert_attention(out[:at], (want[0][:at], want[1][:at]), f"step {step}")
        assert (out[at:] == 7).all()
        if all(n <= 1 for n in new):  # a step of single tokens: the decode call gives the same
            pick = [int(start[g]) for g in range(G)]
            qd = q[[min(i, T - 1) for i in pick]].contiguous()
            one = torch.empty(G, H * 128, dtype=torch.float16, device="cuda")
            ops.paged_decode_attention(one, qd, ck, cv, kn, vn, R, table, lens, page, H, Hkv, bits, ws)
            pu.assert_attention(one, pu.attention(qd, ck, cv, kn, vn, R, table, held, list(range(G + 1)), page, H, Hkv, bits))
