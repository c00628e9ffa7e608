"""Calls at the edges of what the K/V cache and its attention allow, on a B200: refused steps, damaged tables, far ranges, long lists, other
streams.  Tolerances as in test_gpu_kv_cache.py."""
import math
import random

import numpy as np
import pytest

from tests import kv_model
from tests.test_gpu_kv_cache import _build, _check_rows, _t

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx(capi):
    c = capi.Context(0)
    c.use_torch_stream()
    yield c
    c.close()


def _same(a, b):
    return bool(((a == b) | ((a != a) & (b != b))).all())


# ---- pages ----


def test_rows_of_a_refused_step_are_not_stored(capi, ctx):
    """Too few pages, or a list that is unsound: the append behind it, and the steps behind that, leave cache and rows as they were until
    the error has been returned; then the step can be made again."""
    import torch

    cache = _build(capi, "f16", [20, 33, 0], 1, 64, 16, 1, spare=2, max_tokens=200)
    rope = capi.Rope()
    x = torch.randn((90, 64), device="cuda")
    seqs, cu = _t([0, 1]), _t([0, 30, 90])
    for bad, code in ((lambda: ctx.kv_reserve(cache, seqs, cu), capi.ERR_NOMEM), (lambda: ctx.kv_reserve(cache, _t([0, 0])), capi.ERR_ARG)):
        before = [t.clone() for t in (cache.k, cache.v, cache.table, cache.lens, cache.refs)]
        out = torch.full_like(x, 2.0)
        bad()
        ctx.rope_kv_append(cache, 0, x, x, x, seqs, cu, rope, q_out=out)
        ctx.kv_reserve(cache, _t([0]))  # the next step of a loop that does not look
        ctx.rope_kv_append(cache, 0, x[:1], x[:1], x[:1], _t([0]), None, rope, q_out=out[:1])
        with pytest.raises(capi.NhbError) as e:
            ctx.sync()
        assert e.value.code == code
        assert all(_same(a, b) for a, b in zip(before, (cache.k, cache.v, cache.table, cache.lens, cache.refs))) and (out == 2.0).all()
    ctx.kv_reserve(cache, _t([0]))
    ctx.rope_kv_append(cache, 0, x[:1], x[:1], x[:1], _t([0]), None, None)
    ctx.sync()
    assert cache.lens.tolist() == [21, 33, 0]
    assert torch.equal(cache.v[0, cache.table[0, 1].long(), 0, 4], x[0].half())


def test_a_fork_of_a_damaged_table_changes_nothing(capi, ctx):
    """A page number that is none, in a page to be shared or in the one to be copied, of one parent among several: all or nothing."""
    import torch

    cache = _build(capi, "bf16", [40, 0, 33, 0, 0, 7], 2, 64, 16, 1, spare=6, max_tokens=64)
    for column, number in ((0, 99), (1, -5), (2, 1 << 30), (0, -1)):
        for deep in (False, True):
            good = cache.table[0, column].item()
            cache.table[0, column] = number
            before = [t.clone() for t in (cache.table, cache.lens, cache.refs, cache.k, cache.v)]
            ctx.kv_fork(cache, _t([2, 0, 0]), _t([1, 3, 4]), deep=deep)
            with pytest.raises(capi.NhbError) as e:
                ctx.sync()
            assert e.value.code == capi.ERR_ARG
            assert all(_same(a, b) for a, b in zip(before, (cache.table, cache.lens, cache.refs, cache.k, cache.v))), (column, number, deep)
            cache.table[0, column] = good
    cache.table[0, 3] = 99  # behind the last page: no part of the sequence
    ctx.kv_fork(cache, _t([0, -1, 2, 0]), _t([3, -1, 1, 4]))
    ctx.sync()
    assert cache.lens.tolist() == [40, 33, 33, 40, 40, 7] and cache.table[4, :2].tolist() == cache.table[0, :2].tolist() and cache.table[4, 3] == -1
    assert cache.refs[cache.table[0, 0].long()] == 3


# ---- ranges ----


def _both_attentions(capi, ctx, cache, q, scale, heads, d, kind, n):
    """The prompt call over all rows and the decode call of the last, against the formula with the usual tolerances."""
    out = ctx.attn_prompt(cache, 0, q, _t([0]), _t([0, n]), scale)
    last = ctx.attn_decode(cache, 0, q[n - 1 :], _t([0]), scale)
    ctx.sync()
    _check_rows(cache, q.reshape(n, heads, d), out.reshape(n, heads, d), [0], [0, n], scale, kind, what="prompt")
    _check_rows(cache, q[n - 1 :].reshape(1, heads, d), last.reshape(1, heads, d), [0], [0, 1], scale, kind, what="decode")


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("size, q_size, scale", [(1e35, 1.0, 3e-37), (5e37, 1e-3, 5e-37), (1e-30, 1e3, 3e25), (1e-36, 1e9, 3e25), (1e-36, 1e-2, 3e36)])
def test_bf16_keys_of_any_size(capi, ctx, d, size, q_size, scale):
    """Scores of a few units from keys and queries far from 1: what f32 holds is held."""
    n, heads = 300, 4
    cache = _build(capi, "bf16", [n], 2, d, 32, 9)
    cache.k.mul_(size)
    q = (cache.k.new_empty((n, heads * d)).float().normal_()) * q_size
    _both_attentions(capi, ctx, cache, q, scale, heads, d, "bf16", n)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("size", [1e35, 1e-36])
def test_bf16_values_of_any_size(capi, ctx, d, size):
    """Sums of 300 weights times values that f32 holds, also behind a shared prefix."""
    n, heads = 300, 4
    cache = _build(capi, "bf16", [n, n], 2, d, 32, 9)
    cache.v.mul_(size)
    q = cache.k.new_empty((n, heads * d)).float().normal_()
    scale = 1.0 / math.sqrt(d)
    _both_attentions(capi, ctx, cache, q, scale, heads, d, "bf16", n)
    cache.table[1, :8] = cache.table[0, :8]
    out = ctx.attn_decode(cache, 0, q[:2], _t([1, 0]), scale, shared=256)
    ctx.sync()
    _check_rows(cache, q[:2].reshape(2, heads, d), out.reshape(2, heads, d), [1, 0], [0, 1, 2], scale, "bf16", what="shared")


# ---- lists ----


def test_rows_that_two_entries_claim_are_reported(capi, ctx):
    """cu falls behind a padding entry, so that two sequences claim the same rows: more tiles than the call has rows for, in a short and in a
    long list.  Offsets of padding entries alone may be anything."""
    import torch

    cache = _build(capi, "f16", [2000, 2000], 2, 64, 16, 4)
    q = torch.randn((2000, 8 * 64), device="cuda")
    for pad in (20, 700):
        ctx.attn_prompt(cache, 0, q, _t([0, -1] * pad + [1]), _t([0, 2000] * (pad + 1)), 0.125)
        with pytest.raises(capi.NhbError) as e:
            ctx.sync()
        assert e.value.code == capi.ERR_ARG
        seqs, cu = [0] + [-1] * pad + [1], [0, 1000] + [5] * (pad - 1) + [1000, 2000]
        out = ctx.attn_prompt(cache, 0, q, _t(seqs), _t(cu), 0.125)
        ctx.sync()
        _check_rows(cache, q.reshape(-1, 8, 64), out.reshape(-1, 8, 64), [0, 1], [0, 1000, 2000], 0.125, "f16")


@pytest.mark.parametrize("n, two", [(1500, False), (641, True), (1281, False), (640, False)])
def test_prompts_of_more_entries_than_a_block_has_threads(capi, ctx, n, two):
    """The list is looked at in rounds of 640 entries: padding, entries without rows, of one row and of several tiles, at the rounds' borders
    too, and one that is unsound, which is reported while the others are computed."""
    import torch

    r = random.Random(n)
    heads, kv_heads, d, page = (16, 2, 64, 16) if two else (4, 2, 64, 16)
    new = [r.choice((0, 1, 1, 2, 5)) for _ in range(n)]
    for i in (0, 1, 638, 639, 640, 1279, 1280, n - 1):
        if i < n:
            new[i] = 3
    new[min(700, n // 2)] = 700 if not two else 3000
    pads = set(r.sample(range(2, n - 2), n // 8)) - {638, 639, 640, 1279, 1280, min(700, n // 2)}
    lens = [c + r.choice((0, 0, 1, 30)) for c in new]
    cache = _build(capi, "f16", lens, kv_heads, d, page, 3)
    seqs = [-1 if i in pads else i for i in range(n)]
    cu = [0]
    for c in new:
        cu.append(cu[-1] + c)
    M = cu[-1] + 1
    q = torch.randn((M, heads * d), device="cuda")
    live = torch.zeros(M, dtype=torch.bool)
    for i, s in enumerate(seqs):
        if s != -1:
            live[cu[i] : cu[i + 1]] = True
    live = live.cuda()
    bad = next(i for i in range(n // 3, n) if seqs[i] != -1 and new[i] > 0 and new[i] < 6)
    for unsound in (None, n + 5):
        listed = list(seqs)
        if unsound is not None:
            listed[bad] = unsound
        out = torch.full_like(q, 3.25)
        ctx.attn_prompt(cache, 0, q, _t(listed), _t(cu), 0.125, out=out)
        if unsound is None:
            ctx.sync()
        else:
            with pytest.raises(capi.NhbError) as e:
                ctx.sync()
            assert e.value.code == capi.ERR_ARG
            listed[bad] = -1  # its rows stay as they are, like padding
            live[cu[bad] : cu[bad + 1]] = False
        _check_rows(cache, q.reshape(M, heads, d), out.reshape(M, heads, d), listed, cu, 0.125, "f16", what=(n, unsound))
        assert (out[~live] == 3.25).all()


@pytest.mark.parametrize("kind, d, page, heads, kv_heads", [("f16", 128, 64, 32, 8), ("bf16", 128, 32, 6, 2), ("f16", 64, 16, 7, 1), ("bf16", 64, 128, 4, 4)])
def test_a_few_rows_behind_a_long_context(capi, ctx, kind, d, page, heads, kv_heads):
    """Drafts to be verified, and a short turn, behind thousands of cached tokens."""
    import torch

    lens = [(9000, 4), (4321, 1), (2500, 16), (6001, 7)]
    cache = _build(capi, kind, [a + b for a, b in lens], kv_heads, d, page, d + page)
    cu = [0, 4, 5, 21, 28]
    q = torch.randn((28, heads * d), device="cuda") * 1.5
    scale = 1.0 / math.sqrt(d)
    out = ctx.attn_prompt(cache, 0, q, _t([0, 1, 2, 3]), _t(cu), scale)
    ctx.sync()
    _check_rows(cache, q.reshape(28, heads, d), out.reshape(28, heads, d), [0, 1, 2, 3], cu, scale, kind)


def test_append_finds_its_entry_in_a_long_list(capi, ctx):
    """600 list entries (the search goes round beyond 256), one row each, none, or many; a CTA takes one token."""
    import torch

    r = random.Random(5)
    n, d, kv_heads, heads, page = 600, 64, 2, 3, 16
    new = [r.choice((0, 1, 1, 2, 19)) for _ in range(n)]
    for i in (0, 255, 256, 257, 511, 512, n - 1):
        new[i] = 2
    seqs = r.sample(range(n), n)
    for i in r.sample(range(1, n - 1), 40):
        if i not in (255, 256, 257, 511, 512):
            seqs[i] = -1
    cu = np.concatenate([[0], np.cumsum(new)]).tolist()
    M = cu[-1] + 2
    cache = capi.KvCache.empty(1, 2 * n + 100, kv_heads, d, n, 64, page)
    ctx.kv_reserve(cache, _t(seqs), _t(cu))
    q, k, v = (torch.randn((M, h * d), device="cuda") for h in (heads, kv_heads, kv_heads))
    out = ctx.rope_kv_append(cache, 0, q, k, v, _t(seqs), _t(cu), capi.Rope(1e4), q_out=torch.full_like(q, 4.0))
    ctx.sync()
    entry = [(i, t - cu[i]) for i in range(n) for t in range(cu[i], cu[i + 1])]
    live = torch.tensor([seqs[i] != -1 for i, _ in entry] + [False, False]).cuda()
    pos = torch.tensor([p for i, p in entry if seqs[i] != -1]).cuda()
    which = torch.tensor([seqs[i] for i, p in entry if seqs[i] != -1]).cuda()
    turn = lambda x, h: kv_model.rotate(x[live].reshape(-1, h, d), pos, 1e4, "pairs", d)  # noqa: E731
    assert (out[live].double() - turn(q, heads).reshape(len(pos), -1)).abs().max().item() <= 10 * 2.0**-21 and (out[~live] == 4.0).all()
    ids = cache.table[which, pos // page].long()
    got_k, got_v = cache.k[0][ids, :, pos % page].double(), cache.v[0][ids, :, pos % page].double()
    want_k, want_v = turn(k, kv_heads), v[live].reshape(-1, kv_heads, d).double()
    assert ((got_k - want_k).abs() <= want_k.abs() * 2.0**-11 + 10 * 2.0**-21).all() and ((got_v - want_v).abs() <= want_v.abs() * 2.0**-11 + 2.0**-25).all()


# ---- streams ----


def _cudart():
    """The CUDA runtime that torch has loaded."""
    import ctypes as C

    import torch  # noqa: F401  (loads it)

    rt = C.CDLL("libcudart.so.12")
    for name, args in (("cudaStreamCreate", [C.c_void_p]), ("cudaStreamDestroy", [C.c_void_p]), ("cudaStreamBeginCapture", [C.c_void_p, C.c_int]),
                       ("cudaStreamEndCapture", [C.c_void_p, C.c_void_p]), ("cudaGraphDestroy", [C.c_void_p])):
        getattr(rt, name).argtypes, getattr(rt, name).restype = args, C.c_int
    return rt


def _stream(rt):
    import ctypes as C

    s = C.c_void_p()
    assert rt.cudaStreamCreate(C.byref(s)) == 0
    return s.value


def test_streams_that_end_between_calls(capi):
    """A stream may end after nhb_sync, or once another one has been named; what still runs on it is waited for, also where the next stream is
    given its handle."""
    import torch

    rt = _cudart()
    cache = _build(capi, "f16", [9000, 2000, 100], 8, 128, 64, 2)
    q = torch.randn((3, 32 * 128), device="cuda")
    seqs = _t([0, 1, 2])
    outs = [torch.zeros_like(q) for _ in range(24)]
    with capi.Context(0) as ctx:
        torch.cuda.synchronize()
        ref = torch.zeros_like(q)
        torch.cuda.synchronize()
        ctx.attn_decode(cache, 0, q, seqs, 0.09, out=ref)
        ctx.sync()
        for i, out in enumerate(outs):
            s = _stream(rt)
            ctx.set_stream(s)
            for _ in range(3):
                ctx.attn_decode(cache, 0, q, seqs, 0.09, out=out)
            if i % 3 == 0:
                ctx.sync()
                assert rt.cudaStreamDestroy(s) == 0
                ctx.set_stream(None)
            else:
                ctx.set_stream(None)
                assert rt.cudaStreamDestroy(s) == 0
            if i % 2:
                ctx.attn_decode(cache, 0, q, seqs, 0.09, out=out)
        ctx.sync()
        torch.cuda.synchronize()
        assert all(torch.equal(o, ref) for o in outs)


def test_a_capture_open_elsewhere_does_not_hold_the_context_on_the_legacy_stream(capi):
    """From the legacy stream to a blocking stream that is being captured, and back."""
    import ctypes as C

    import torch

    rt = _cudart()
    cache = _build(capi, "f16", [900, 20], 2, 64, 16, 2)
    q = torch.randn((2, 8 * 64), device="cuda")
    seqs = _t([0, 1])
    ref, out, last = (torch.zeros_like(q) for _ in range(3))
    s, graph = _stream(rt), C.c_void_p()
    with capi.Context(0) as ctx:
        ctx.set_stream(1)
        ctx.attn_decode(cache, 0, q, seqs, 0.125, out=ref)
        assert rt.cudaStreamBeginCapture(s, 1) == 0
        try:
            ctx.set_stream(s)
            ctx.attn_decode(cache, 0, q, seqs, 0.125, out=out)
        finally:
            assert rt.cudaStreamEndCapture(s, C.byref(graph)) == 0
        ctx.attn_decode(cache, 0, q, seqs, 0.125, out=last)
        ctx.set_stream(None)
        ctx.attn_decode(cache, 0, q, seqs, 0.125, out=last)
        ctx.sync()
        ctx.set_stream(1)
        ctx.sync()
        torch.cuda.synchronize()
        assert torch.equal(ref, last) and (out == 0).all()  # captured, not run
    assert rt.cudaGraphDestroy(graph) == 0 and rt.cudaStreamDestroy(s) == 0


def test_new_outputs_of_a_context_on_another_stream(capi):
    """torch fills a new output with zeros on its own stream, here behind a long product; the context's rows must not come first."""
    import torch

    cache = _build(capi, "f16", [90, 20], 2, 64, 16, 2)
    q, kv = torch.randn((2, 8 * 64), device="cuda"), torch.randn((2, 128), device="cuda")
    seqs, cu = _t([0, 1]), _t([0, 1, 2])
    a = torch.randn((8192, 8192), device="cuda")
    side = torch.cuda.Stream()
    for stream in (None, side.cuda_stream):
        with capi.Context(0) as ctx:
            ctx.set_stream(stream)
            calls = [lambda **o: ctx.attn_decode(cache, 0, q, seqs, 0.125, **o), lambda **o: ctx.attn_prompt(cache, 0, q, seqs, cu, 0.125, **o),
                     lambda **o: ctx.rope_kv_append(cache, 0, q, kv, kv, seqs, **{{"out": "q_out"}[k]: v for k, v in o.items()})]
            for call in calls:
                ref = torch.zeros_like(q)
                torch.cuda.synchronize()
                call(out=ref)
                ctx.sync()
                a @ a  # some 15 ms of torch's stream
                got = call()
                ctx.sync()
                torch.cuda.synchronize()
                assert torch.equal(got, ref) and (got != 0).any()


def test_graphs_and_eager_calls_on_streams_in_turn(capi):
    """One workspace: replays of two graphs and eager calls, each on another stream than the one before, none of them waited for."""
    import torch

    cache = _build(capi, "f16", [5000, 3000, 100], 8, 128, 64, 2)
    q = torch.randn((3, 32 * 128), device="cuda")
    seqs, fewer = _t([0, 1, 2]), _t([1, 2, 0])
    streams = [torch.cuda.Stream() for _ in range(3)]
    ref, other, a, b, c = (torch.zeros_like(q) for _ in range(5))
    torch.cuda.synchronize()
    with capi.Context(0) as ctx:
        ctx.attn_decode(cache, 0, q, seqs, 0.09, out=ref)
        ctx.attn_decode(cache, 0, q, fewer, 0.09, out=other)
        ctx.sync()
        graphs = []
        for which, out in ((seqs, a), (fewer, b)):
            ctx.graph_begin()
            ctx.attn_decode(cache, 0, q, which, 0.09, out=out)
            graphs.append(ctx.graph_end())
        for i in range(30):
            ctx.set_stream(streams[i % 3].cuda_stream)
            if i % 4 == 3:
                ctx.attn_decode(cache, 0, q, seqs, 0.09, out=c)
            else:
                graphs[i % 2].launch()
        ctx.sync()
        torch.cuda.synchronize()
        assert torch.equal(a, ref) and torch.equal(b, other) and torch.equal(c, ref)
        for g in graphs:
            g.free()


def test_compact_reports_a_length_it_cannot_follow(capi, ctx):
    """The pages of such a sequence may move without its table: the caller has to know."""
    cache = _build(capi, "f16", [40, 33, 16, 50], 1, 64, 16, 1, spare=6, max_tokens=64)
    for length in (65, -1, 1 << 30):
        cache.lens[1] = length
        ctx.kv_compact(cache)
        with pytest.raises(capi.NhbError) as e:
            ctx.sync()
        assert e.value.code == capi.ERR_ARG
    cache.lens[1] = 0
    ctx.kv_compact(cache)
    ctx.sync()


def test_compact_leaves_a_page_that_nobody_counts_where_it_is(capi, ctx):
    """A table that holds a page whose count is zero, behind the pages in use: no move belongs to it.  It is reported and keeps its number."""
    for behind in (1, 4):
        cache = _build(capi, "f16", [40, 33, 16, 50], 1, 64, 16, 1, spare=6, max_tokens=64)
        ctx.kv_free(cache, _t([0]))
        ctx.kv_compact(cache)
        ctx.sync()
        page = int((cache.refs > 0).sum()) + behind  # free
        cache.refs[cache.table[1, 0].long()] = 0
        cache.table[1, 0] = page
        others = cache.table[2:4].clone()
        ctx.kv_compact(cache)  # one gap is closed by the last page in use
        with pytest.raises(capi.NhbError) as e:
            ctx.sync()
        assert e.value.code == capi.ERR_ARG and cache.table[1, 0].item() == page
        assert int((cache.table[2:4] != others).sum()) <= 1
