"""Refusals of the paged calls: every one happens before anything is enqueued, so no GPU is needed."""
import ctypes as C

import pytest

import triebwerk_b200 as tq

P = C.c_void_p(1 << 20)  # never followed: the call is refused first
ODD = C.c_void_p((1 << 20) + 2)


def plan(**kw):
    a = dict(table=P, stride=8, width=8, free=P, count=P, count_out=P, pages=16, page=32, context=P, new=P, finished=None, G=4, lens=P, start=P, slots=P,
             positions=None, T=4)
    a.update(kw)
    return tq.lib().tq_page_plan(*a.values(), None)


def rows(name, **kw):
    a = dict(ck=P, kn=P, cv=P, vn=P, k=P, v=P, R=P, slots=P, rows=64, T=2, Hkv=8, D=128, stride=1024, bits=4)
    a.update(kw)
    if name == "tq_paged_read":
        a = {k: a[k] for k in ("k", "v", "ck", "kn", "cv", "vn", "R", "slots", "rows", "T", "Hkv", "D", "stride", "bits")}
    return getattr(tq.lib(), name)(*a.values(), None)


def attention(**kw):
    a = dict(out=P, q=P, ck=P, cv=P, kn=P, vn=P, R=P, table=P, stride=8, width=8, lens=P, pages=16, page=32, G=4, H=16, Hkv=8, D=128, qs=2048, os=2048, bits=4,
             ws=P, bytes=1 << 30)
    a.update(kw)
    return tq.lib().tq_paged_decode_attention(*a.values(), None)


@pytest.mark.parametrize("change, status", [
    (dict(page=16), -4), (dict(page=48), -4), (dict(page=0), -4), (dict(page=131072), -4), (dict(width=0), -1), (dict(stride=7), -1), (dict(pages=0), -1),
    (dict(pages=1 << 27), -4), (dict(width=1 << 26, stride=1 << 26), -4), (dict(table=None), -1), (dict(free=None), -1), (dict(count=None), -1),
    (dict(count_out=None), -1), (dict(context=None), -1), (dict(new=None), -1), (dict(lens=None), -1), (dict(start=None), -1), (dict(slots=None), -1),
    (dict(G=0), -1), (dict(T=-1), -1)])
def test_plan_refuses(change, status):
    assert plan(**change) == status


@pytest.mark.parametrize("name", ["tq_paged_append", "tq_paged_read"])
@pytest.mark.parametrize("change, status", [
    (dict(D=64), -4), (dict(bits=0), -1), (dict(bits=3), -1), (dict(Hkv=0), -1), (dict(rows=0), -1), (dict(rows=1 << 31), -4), (dict(stride=1016), -1),
    (dict(stride=1028), -1), (dict(T=-1), -1), (dict(T=1 << 28), -4), (dict(ck=None), -1), (dict(kn=None), -1), (dict(cv=None), -1), (dict(vn=None), -1),
    (dict(k=None), -1), (dict(v=None), -1), (dict(R=None), -1), (dict(slots=None), -1), (dict(ck=ODD), -1), (dict(k=ODD), -1), (dict(v=ODD), -1),
    (dict(R=ODD), -1)])
def test_rows_refuse(name, change, status):
    assert rows(name, **change) == status


@pytest.mark.parametrize("name", ["tq_paged_append", "tq_paged_read"])
def test_no_tokens_is_no_work(name):
    assert rows(name, T=0, k=None, v=None, slots=None) == 0


def prefill(**kw):
    a = dict(out=P, q=P, ck=P, cv=P, kn=P, vn=P, R=P, table=P, stride=8, width=8, lens=P, start=P, pages=16, page=32, T=7, G=4, H=16, Hkv=8, D=128, qs=2048,
             os=2048, bits=4, ws=P, bytes=1 << 30)
    a.update(kw)
    return tq.lib().tq_paged_prefill_attention(*a.values(), None)


@pytest.mark.parametrize("change, status", [
    (dict(start=None), -1), (dict(T=-1), -1), (dict(H=258, Hkv=2, qs=258 * 128, os=258 * 128), -4), (dict(bytes=1000), -3), (dict(ws=None), -3), (dict(lens=None), -1),
    (dict(table=None), -1), (dict(page=24), -4), (dict(G=0), -1), (dict(bits=0), -1), (dict(q=ODD), -1), (dict(qs=2044), -1),
    (dict(G=65536, bytes=1 << 33), -4), (dict(T=1 << 27), -4)])
def test_prefill_refuses(change, status):
    assert prefill(**change) == status


def test_prefill_of_no_tokens_is_no_work():
    assert prefill(T=0) == 0


@pytest.mark.parametrize("change, status", [
    (dict(page=16), -4), (dict(page=96), -4), (dict(D=64), -4), (dict(bits=0), -1), (dict(bits=8), -1), (dict(G=0), -1), (dict(H=15), -1), (dict(Hkv=0), -1),
    (dict(H=0), -1), (dict(qs=2040), -1), (dict(qs=2052), -1), (dict(os=2047), -1), (dict(stride=4), -1), (dict(width=0), -1), (dict(pages=0), -1),
    (dict(pages=1 << 26), -4), (dict(out=None), -1), (dict(q=None), -1), (dict(ck=None), -1), (dict(cv=None), -1), (dict(kn=None), -1), (dict(vn=None), -1),
    (dict(R=None), -1), (dict(table=None), -1), (dict(lens=None), -1), (dict(ws=None), -3), (dict(ws=ODD), -3), (dict(bytes=1000), -3), (dict(q=ODD), -1),
    (dict(out=ODD), -1), (dict(kn=ODD), -1), (dict(G=65536, bytes=1 << 33), -4)])
def test_decode_refuses(change, status):
    assert attention(**change) == status


def test_workspace_sizes():
    f = tq.lib().tq_paged_workspace_bytes
    assert f(1, 0, 16) == 0 and f(-1, 1, 16) == 0 and f(1, 1, 0) == 0
    assert 0 < f(4, 4, 16) < f(64, 64, 16) < f(64, 64, 32)


# (nothing is launched: what is refused is the overlap, before the device is asked for anything)
@pytest.mark.parametrize("out, q, qs, os", [(0, 0, 2048, 2048), (2048, 0, 2048, 2048), (0, 2048 * 2, 2048, 2048), (2040, 0, 4096, 4096), (4096 * 2 - 8, 0, 4096, 4096), (64, 0, 2048, 4096)])
@pytest.mark.parametrize("call", [attention, prefill])
def test_results_over_queries_are_refused(call, out, q, qs, os):
    at = lambda halves: C.c_void_p((1 << 20) + 2 * halves)  # noqa: E731
    assert call(out=at(out), q=at(q), qs=qs, os=os) == -1


def test_results_over_results_are_refused():
    for k, v, stride in ((0, 0, 1024), (0, 1024, 1024), (0, 512, 2048), (1536, 0, 2048)):
        assert rows("tq_paged_read", k=C.c_void_p((1 << 20) + 2 * k), v=C.c_void_p((1 << 20) + 2 * v), stride=stride) == -1


# Arrays in their order of address, none touching the next: 1 MiB apart, each smaller than that.
def apart(names):
    return {n: C.c_void_p((i + 1) << 20) for i, n in enumerate(names)}


def shared(a, name, other, size):
    """`name` on the last bytes of `other`, which has `size` (where its own alignment lets it begin)."""
    to = 256 if name == "ws" else 16
    return dict(a, **{name: C.c_void_p(a[other].value + (size - 1) // to * to)})


PLAN = dict(table=4 * 32, free=64, count=4, count_out=4, context=16, new=16, finished=4, lens=16, start=20, slots=32, positions=16)
PLAN_READ = ("count", "context", "new", "finished")


@pytest.mark.parametrize("name", PLAN)
@pytest.mark.parametrize("other", PLAN)
def test_plan_refuses_arrays_that_share_memory(name, other):
    # (count and count_out, context and lens may be the same array: not in part, as here, but where an array has 16 bytes or fewer)
    if name == other or (name in PLAN_READ and other in PLAN_READ) or {name, other} in ({"count", "count_out"}, {"context", "lens"}):
        return
    assert plan(**shared(apart(PLAN), name, other, PLAN[other])) == -1


def test_plan_refuses_lengths_that_are_the_context_in_part():
    a = apart(PLAN)
    a["lens"] = C.c_void_p(a["context"].value + 4)
    assert plan(**a) == -1


ROWS = dict(ck=64 * 512, kn=64 * 16, cv=64 * 512, vn=64 * 16, k=4096, v=4096, R=32768, slots=16)


@pytest.mark.parametrize("call, written", [("tq_paged_append", ("ck", "kn", "cv", "vn")), ("tq_paged_read", ("k", "v"))])
@pytest.mark.parametrize("name", ROWS)
@pytest.mark.parametrize("other", ROWS)
def test_rows_refuse_arrays_that_share_memory(call, written, name, other):
    if name != other and (name in written or other in written):
        assert rows(call, **shared(apart(ROWS), name, other, ROWS[other])) == -1


ATTENTION = dict(out=4 * 4096, q=4 * 4096, ck=512 * 512, cv=512 * 512, kn=512 * 16, vn=512 * 16, R=32768, table=4 * 32, lens=16, ws=4 * 16 * 132 * 4)


@pytest.mark.parametrize("call, arrays", [(attention, ATTENTION), (prefill, dict(ATTENTION, out=7 * 4096, q=7 * 4096, start=20))])
@pytest.mark.parametrize("written", ["out", "ws"])
@pytest.mark.parametrize("other", [*ATTENTION, "start"])
def test_attentions_refuse_arrays_that_share_memory(call, arrays, written, other):
    if other == written or other not in arrays:
        return
    a = apart(arrays)
    a["ws"] = C.c_void_p(64 << 20)
    assert call(**shared(a, other, written, arrays[written])) == -1
    if written == "out":
        assert call(**shared(a, written, other, arrays[other])) == -1


# (an address that is no multiple of the element's size would fault on the GPU)
@pytest.mark.parametrize("name, off", [(n, 2) for n in PLAN if n not in ("finished", "slots")] + [("slots", 4)])
def test_plan_refuses_addresses_that_no_element_has(name, off):
    a = apart(PLAN)
    assert plan(**dict(a, **{name: C.c_void_p(a[name].value + off)})) == -1


@pytest.mark.parametrize("call", ["tq_paged_append", "tq_paged_read"])
@pytest.mark.parametrize("name, off", [("ck", 8), ("cv", 8), ("kn", 1), ("vn", 1), ("k", 8), ("v", 8), ("R", 8), ("slots", 4)])
def test_rows_refuse_addresses_that_no_element_has(call, name, off):
    a = apart(ROWS)
    assert rows(call, **dict(a, **{name: C.c_void_p(a[name].value + off)})) == -1


@pytest.mark.parametrize("call, arrays", [(attention, ATTENTION), (prefill, dict(ATTENTION, start=20))])
@pytest.mark.parametrize("name, off", [(n, 8) for n in ("out", "q", "ck", "cv", "kn", "vn", "R")] + [("table", 2), ("lens", 2), ("start", 2)])
def test_attentions_refuse_addresses_that_no_element_has(call, arrays, name, off):
    if name in arrays:
        a = dict(apart(arrays), ws=C.c_void_p(64 << 20))
        assert call(**dict(a, **{name: C.c_void_p(a[name].value + off)})) == -1


def test_no_query_rows_need_no_arrays():
    # (an empty tensor has no address)
    assert prefill(T=0, out=None, q=None) == 0
    assert prefill(out=None) == -1 and prefill(q=None) == -1
