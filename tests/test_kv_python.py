"""The Python layer of the K/V cache: what it hands to the library, and what it refuses (no GPU needed: nothing here is launched)."""
import pytest


class Factors:
    """Looks like an f32 tensor on a GPU."""

    def __init__(self, n, ptr, device=0):
        import torch

        self.dtype, self.shape, self.ptr, self.device_index = torch.float32, (n,), ptr, device
        self.is_cuda = True

    def dim(self):
        return len(self.shape)

    def is_contiguous(self):
        return True

    def data_ptr(self):
        return self.ptr

    def get_device(self):
        return self.device_index


def test_a_rotation_is_what_was_last_assigned_to_it(capi):
    rope = capi.Rope(10000.0, factors=Factors(64, 4096))

    def now(head_dim=128):
        s = rope.ref(head_dim)._obj
        return s.base, s.dims, s.style, s.factors

    assert now() == (10000.0, 128, 0, 4096) and now(64) == (10000.0, 64, 0, 4096)
    assert rope.ref(128) is rope.ref(128)  # made once
    rope.base = 5e5
    assert now() == (5e5, 128, 0, 4096)
    rope.factors = Factors(64, 8192)
    assert now() == (5e5, 128, 0, 8192) and now(64) == (5e5, 64, 0, 8192)
    rope.dims, rope.style = 32, "halves"
    assert now() == (5e5, 32, 1, 8192)
    rope.factors = None
    assert now() == (5e5, 32, 1, None)
    rope.factors = Factors(15, 8192)
    with pytest.raises(capi.NhbError):
        rope.ref(128)
    rope.factors, rope.style = None, "spiral"
    with pytest.raises(capi.NhbError):
        rope.ref(128)


class Rows:
    """Looks like f32 rows on GPU 0."""

    def __init__(self, rows, width, ptr, stride=None):
        import torch

        self.dtype, self.shape, self.ptr, self.strides = torch.float32, (rows, width), ptr, (stride or width, 1)

    def stride(self):
        return self.strides

    def data_ptr(self):
        return self.ptr

    def get_device(self):
        return 0


class List:
    """Looks like an int32 tensor on GPU 0."""

    def __init__(self, *shape, ptr=1 << 20):
        import torch

        self.dtype, self.shape, self.ptr = torch.int32, shape, ptr

    def is_contiguous(self):
        return True

    def dim(self):
        return len(self.shape)

    def numel(self):
        n = 1
        for x in self.shape:
            n *= x
        return n

    def data_ptr(self):
        return self.ptr

    def get_device(self):
        return 0


def _context(capi):
    """A context of GPU 0 without a handle: calls get as far as the library's own check of it, which comes last."""
    ctx = capi.Context.__new__(capi.Context)
    ctx.handle, ctx.device = None, 0
    return ctx


def _cache(capi, max_seqs=4):
    import ctypes as C

    cache = capi.KvCache.__new__(capi.KvCache)
    p = 1 << 20
    struct = capi.KvCacheStruct(p, 2 * p, 3 * p, 4 * p, 5 * p, 1, 8, 2, 16, 64, max_seqs, 4, 0)
    cache.__dict__.update(kv_heads=2, head_dim=64, device=0, struct=struct, ref=C.byref(struct))
    return cache


def _refused(capi, text, call, *args, **kw):
    with pytest.raises(capi.NhbError) as e:
        call(*args, **kw)
    assert e.value.code == capi.ERR_ARG and text in str(e.value), e.value


def test_factors_on_another_gpu_are_refused(capi):
    ctx, cache = _context(capi), _cache(capi)
    q, k, v, out = (Rows(2, w, (i + 1) << 24) for i, w in enumerate((256, 128, 128, 256)))
    here, there = capi.Rope(factors=Factors(32, 4096)), capi.Rope(factors=Factors(32, 4096, device=1))
    _refused(capi, "null context", ctx.rope_kv_append, cache, 0, q, k, v, List(2), rope=here, q_out=out)  # all else is in order
    _refused(capi, "another GPU", ctx.rope_kv_append, cache, 0, q, k, v, List(2), rope=there, q_out=out)


def test_lists_count_all_their_entries(capi, monkeypatch):
    """Whatever the shape of a list, as many entries reach the library as it holds."""
    seen = {}

    class Library:
        def __getattr__(self, name):
            return lambda *args: seen.setdefault(name, []).append(args) or 0

    monkeypatch.setattr(capi, "lib", Library())
    ctx, cache = _context(capi), _cache(capi)
    for shape in ((6,), (1, 6), (6, 1), (2, 3)):
        seen.clear()
        many = List(*shape)
        q, k, v, out = (Rows(6, w, (i + 1) << 24) for i, w in enumerate((256, 128, 128, 256)))
        cu = List(7)
        ctx.kv_reserve(cache, many)
        ctx.kv_reserve(cache, many, cu)
        ctx.kv_free(cache, many)
        ctx.kv_fork(cache, many, List(*shape))
        ctx.rope_kv_append(cache, 0, q, k, v, many, q_out=out)
        ctx.attn_prompt(cache, 0, q, many, cu, 0.1, out=out)
        ctx.attn_decode(cache, 0, q, many, 0.1, out=out)
        counts = [a[4] for a in seen["nhb_kv_reserve"]] + [a[3] for a in seen["nhb_kv_free"]] + [a[4] for a in seen["nhb_kv_fork"]]
        counts += [a[13] for a in seen["nhb_rope_kv_append"]] + [a[9] for a in seen["nhb_attn_prompt"]] + [a[7] for a in seen["nhb_attn_decode"]]
        assert counts == [6] * 7, (shape, counts)
        with pytest.raises(capi.NhbError):
            ctx.kv_reserve(cache, many, List(6))
        with pytest.raises(capi.NhbError):
            ctx.attn_decode(cache, 0, Rows(5, 256, 1 << 24), many, 0.1, out=Rows(5, 256, 2 << 24))


def test_compact_refuses_a_place_without_room(capi):
    """An empty slice has an address, and the number would land behind it."""
    ctx, cache = _context(capi), _cache(capi)
    _refused(capi, "null context", ctx.kv_compact, cache, List(1))
    _refused(capi, "null context", ctx.kv_compact, cache, List())
    _refused(capi, "no room", ctx.kv_compact, cache, List(0))


def test_the_stride_of_one_row_does_not_matter(capi):
    """A single row of a wider buffer, whatever the buffer's row length."""
    ctx, cache = _context(capi), _cache(capi)
    for stride in (256, 260, 261, 1, 0):
        q, out = Rows(1, 256, 1 << 24, stride), Rows(1, 256, 2 << 24, stride)
        k, v = Rows(1, 128, 3 << 24, stride), Rows(1, 128, 4 << 24, stride)
        _refused(capi, "null context", ctx.attn_decode, cache, 0, q, List(1), 0.1, out=out)
        _refused(capi, "null context", ctx.attn_prompt, cache, 0, q, List(1), List(2), 0.1, out=out)
        _refused(capi, "null context", ctx.rope_kv_append, cache, 0, q, k, v, List(1), q_out=q)
    _refused(capi, "rows", ctx.attn_decode, cache, 0, Rows(2, 256, 1 << 24, 261), List(2), 0.1, out=Rows(2, 256, 2 << 24))
    # a row of q, k and v side by side: they do not meet, and a row that does is refused
    q, k, v = Rows(1, 256, 1 << 24, 515), Rows(1, 128, (1 << 24) + 1024, 515), Rows(1, 128, (1 << 24) + 1536, 515)
    _refused(capi, "null context", ctx.rope_kv_append, cache, 0, q, k, v, List(1), q_out=q)
    _refused(capi, "overlap", ctx.rope_kv_append, cache, 0, q, k, v, List(1), q_out=Rows(1, 256, (1 << 24) + 512, 515))


def test_the_tensors_of_a_cache_cannot_be_replaced(capi):
    """The C struct holds their pointers: an assignment would be ignored, and the old memory read after its end."""
    import torch

    cache = _cache(capi)
    for name in ("k", "v", "table", "lens", "refs"):
        t = torch.zeros(3)
        setattr(cache, name, t)
        setattr(cache, name, t)  # what `cache.k *= 2` does
        with pytest.raises(capi.NhbError):
            setattr(cache, name, t.clone())
        assert getattr(cache, name) is t
    cache.note = 1


def test_a_table_whose_size_overflows_is_refused(capi):
    """2^60 pages of 16 tokens are 2^64 tokens, which 64 bits take for none."""
    import ctypes as C

    p = 1 << 20
    for max_pages, page in ((1 << 60, 16), ((1 << 60) + 5, 16), (1 << 57, 128), ((1 << 23) + 1, 128), (1 << 62, 64)):
        struct = capi.KvCacheStruct(p, 2 * p, 3 * p, 4 * p, 5 * p, 1, 8, 2, page, 64, 4, max_pages, 0)
        rc = capi.lib.nhb_kv_free(None, C.byref(struct), p, 1)
        assert rc == capi.ERR_ARG and "out of range" in capi.last_error(), (max_pages, page, capi.last_error())
    struct = capi.KvCacheStruct(p, 2 * p, 3 * p, 4 * p, 5 * p, 1, 8, 2, 128, 64, 4, 1 << 23, 0)
    assert capi.lib.nhb_kv_free(None, C.byref(struct), p, 1) == capi.ERR_ARG and "null context" in capi.last_error()


def test_torchs_stream_is_that_of_the_contexts_gpu(capi, monkeypatch):
    """Asked for by the context's own device, whatever device is current; the same stream is not set twice."""
    current = {0: 0, 1: 7777}
    monkeypatch.setattr(capi, "_current_stream", current.__getitem__)
    for device, handles in ((0, [1, 5555]), (1, [7777, 8888])):
        ctx, sets = _context(capi), []
        ctx.device = device
        monkeypatch.setattr(ctx, "set_stream", lambda h, ctx=ctx, sets=sets: (sets.append(h), setattr(ctx, "stream", h)))
        ctx.use_torch_stream()
        ctx.use_torch_stream()
        current[device] = handles[1]
        ctx.use_torch_stream()
        assert sets == handles
