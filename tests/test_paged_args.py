"""Refusals of the batched-serving entry points: checked on the host, before anything reaches the GPU."""
import ctypes as C

import pytest


def structs(nc):
    cache = nc.PagedCache(k=16, v=16, k_deltas=16, v_deltas=16, dtype=nc.F16, n_pages=8, page_size=16, n_kv_heads=2,
                          d_head=64)
    batch = nc.PagedBatch(n_req=2, max_tokens=4, max_pages=3, max_new=2, max_kv=40, new_len=4096, seq_len=8192,
                          block_table=16, row_start=16, kv_len=64, positions=128, slots=256)
    pool = nc.PagePool(free_pages=16, state=16, n_pages=8, page_size=16)
    return cache, batch, pool


def refused(nc, status, word):
    assert status == -1, status
    assert word in nc.lib().nc_last_error().decode(), nc.lib().nc_last_error()


CACHE = [("k", None, "null"), ("dtype", 2, "dtype"), ("dtype", 4, "dtype"), ("d_head", 96, "head size"),
         ("page_size", 8, "page size"), ("page_size", 48, "page size"), ("page_size", 2048, "page size"),
         ("n_kv_heads", 0, "kv heads"), ("n_pages", 0, "pages"), ("n_pages", 1 << 28, "pages"), ("v", 24, "aligned")]
BATCH = [("n_req", 0, "requests"), ("n_req", 4097, "requests"), ("max_tokens", -1, "rows"), ("max_new", -1, "bounds"),
         ("max_kv", -1, "bounds"), ("max_kv", (1 << 24) + 1, "bounds"), ("max_pages", 2, "pages a request"),
         ("block_table", None, "null table"), ("slots", None, "null table")]


@pytest.mark.parametrize("field,value,word", CACHE)
def test_cache_refusals(nc, field, value, word):
    L = nc.lib()
    cache, batch, _ = structs(nc)
    setattr(cache, field, value)
    q = nc.Tensor(16, None, nc.F16, 4, 256, 512)
    kv = nc.Tensor(16, None, nc.F16, 4, 128, 256)
    size = C.c_size_t()
    refused(nc, L.nc_paged_attn_workspace(C.byref(cache), C.byref(batch), 4, 0, 0, C.byref(size)), word)
    refused(nc, L.nc_paged_attn(C.byref(q), C.byref(cache), C.byref(batch), C.byref(q), 4, 0, 0, None, 0, None), word)
    refused(nc, L.nc_paged_append(C.byref(q), C.byref(kv), C.byref(kv), C.byref(q), C.byref(cache), C.byref(batch), None,
                                  0, 0, None), word)


def test_q8_cache_needs_deltas(nc):
    cache, batch, _ = structs(nc)
    cache.dtype, cache.v_deltas = nc.Q8, None
    size = C.c_size_t()
    refused(nc, nc.lib().nc_paged_attn_workspace(C.byref(cache), C.byref(batch), 4, 0, 0, C.byref(size)), "deltas")


@pytest.mark.parametrize("field,value,word", BATCH)
def test_batch_refusals(nc, field, value, word):
    L = nc.lib()
    cache, batch, pool = structs(nc)
    setattr(batch, field, value)
    size = C.c_size_t()
    refused(nc, L.nc_paged_attn_workspace(C.byref(cache), C.byref(batch), 4, 0, 0, C.byref(size)), word)
    refused(nc, L.nc_paged_plan(C.byref(pool), C.byref(batch), None), word)
    refused(nc, L.nc_paged_commit(C.byref(pool), C.byref(batch), None, None), word)


@pytest.mark.parametrize("field,value,word", [("free_pages", None, "null pool"), ("state", None, "null pool"),
                                              ("page_size", 17, "page size"), ("n_pages", 0, "pages"),
                                              ("n_pages", 1 << 27, "pages")])
def test_pool_refusals(nc, field, value, word):
    L = nc.lib()
    _, batch, pool = structs(nc)
    setattr(pool, field, value)
    refused(nc, L.nc_page_pool_init(C.byref(pool), None), word)
    refused(nc, L.nc_paged_plan(C.byref(pool), C.byref(batch), None), word)


def test_plan_refuses_tables_over_the_lengths(nc):
    L = nc.lib()
    for field in ("kv_len", "row_start", "positions", "slots"):
        for lens in ("seq_len", "new_len"):
            _, batch, pool = structs(nc)
            setattr(batch, field, getattr(batch, lens) + 4)
            refused(nc, L.nc_paged_plan(C.byref(pool), C.byref(batch), None), "over the lengths")


def test_null_structs(nc):
    L = nc.lib()
    cache, batch, pool = structs(nc)
    size = C.c_size_t()
    refused(nc, L.nc_paged_plan(None, C.byref(batch), None), "null pool")
    refused(nc, L.nc_paged_plan(C.byref(pool), None, None), "null batch")
    refused(nc, L.nc_paged_attn_workspace(None, C.byref(batch), 4, 0, 0, C.byref(size)), "null cache")
    refused(nc, L.nc_paged_attn_workspace(C.byref(cache), C.byref(batch), 4, 0, 0, None), "null result")
    batch.seq_len = None
    refused(nc, L.nc_paged_plan(C.byref(pool), C.byref(batch), None), "null lengths")


def test_attention_refusals(nc):
    L = nc.lib()
    cache, batch, _ = structs(nc)
    size = C.c_size_t()
    ok = lambda t=None, **kw: nc.Tensor(**{**dict(data=16, deltas=None, dtype=nc.F16, rows=4, cols=256,  # noqa: E731
                                                  pitch=512), **kw})

    def call(q, out, heads=4, window=0, sink=0, work=None, n=0):
        return L.nc_paged_attn(C.byref(q), C.byref(cache), C.byref(batch), C.byref(out), heads, window, sink, work, n, None)

    refused(nc, call(ok(), ok(), heads=3), "3 heads over 2")
    refused(nc, call(ok(), ok(), heads=0), "heads")
    refused(nc, call(ok(), ok(), window=-1), "window")
    refused(nc, call(ok(), ok(), window=5, sink=-1), "sinks")
    for bad in (dict(rows=3), dict(cols=128), dict(data=None), dict(data=24), dict(pitch=496), dict(pitch=520)):
        refused(nc, call(ok(**bad), ok()), "aligned rows")
        refused(nc, call(ok(), ok(**bad)), "aligned rows")
    refused(nc, call(ok(dtype=nc.F32, pitch=1024), ok()), "dtypes")
    refused(nc, call(ok(), ok(dtype=nc.F32, pitch=1024)), "dtypes")
    batch.max_kv, batch.max_pages = 4096, 256
    nc.check(L.nc_paged_attn_workspace(C.byref(cache), C.byref(batch), 4, 0, 0, C.byref(size)))
    assert size.value > 0
    refused(nc, call(ok(), ok(), work=16, n=size.value - 1), "workspace")
    refused(nc, call(ok(), ok(), work=None, n=size.value), "workspace")
    refused(nc, call(ok(), ok(), work=24, n=size.value), "workspace")


def test_append_refusals(nc):
    L = nc.lib()
    cache, batch, _ = structs(nc)
    row = lambda cols, **kw: nc.Tensor(**{**dict(data=1 << 20, deltas=None, dtype=nc.F16, rows=4, cols=cols,  # noqa: E731
                                                 pitch=2 * cols), **kw})

    def call(q, k, v, out, rope=None, rows=0, half=0):
        r = lambda t: C.byref(t) if t is not None else None  # noqa: E731
        return L.nc_paged_append(r(q), r(k), r(v), r(out), C.byref(cache), C.byref(batch), rope, rows, half, None)

    q, k, out = row(256), row(128), row(256, data=1 << 22)
    refused(nc, call(q, row(64), k, out), "k and v")
    refused(nc, call(q, k, row(128, dtype=nc.F32, pitch=512), out), "k and v")
    refused(nc, call(q, row(128, rows=3), k, out), "k and v")
    refused(nc, call(None, k, k, out), "together")
    refused(nc, call(q, k, k, None), "together")
    refused(nc, call(row(200, pitch=416), k, k, out), "q of 200")
    refused(nc, call(row(256, dtype=nc.F32, pitch=1024), k, k, out), "k's type")
    refused(nc, call(q, k, k, row(256, data=1 << 22, dtype=nc.F32, pitch=1024)), "q_out dtype")
    refused(nc, call(q, k, k, row(256, data=(1 << 20) + 512)), "lies over q")
    refused(nc, call(q, k, k, out, rope=16, rows=0, half=32), "rope table")
    refused(nc, call(q, k, k, out, rope=16, rows=9, half=33), "rope table")
    refused(nc, call(q, k, k, out, rope=16, rows=9, half=-1), "rope table")
    refused(nc, call(q, k, k, out, rope=20, rows=9, half=32), "rope table")


def test_lora_refusals(nc):
    L = nc.lib()
    base = dict(a=16, b=16, scale=16, n_adapters=3, rank=16, k=64, n=100)
    x = nc.Tensor(16, None, nc.F16, 4, 64, 128)
    y = nc.Tensor(16, None, nc.F32, 4, 100, 400)

    def call(x=x, y=y, out=y, n_req=2, max_new=2, adapter=16, **kw):
        lora = nc.Lora(**{**base, **kw})
        return L.nc_lora_add(C.byref(x), C.byref(y), C.byref(lora), adapter, 16, n_req, max_new, C.byref(out), None)

    refused(nc, call(rank=0), "rank")
    refused(nc, call(rank=129), "rank")
    refused(nc, call(k=48), "multiple of 32")
    refused(nc, call(n=0), "adapters")
    refused(nc, call(n_adapters=0), "adapters")
    refused(nc, call(a=None), "null")
    refused(nc, call(scale=None), "null")
    refused(nc, call(adapter=None), "null")
    refused(nc, call(b=24), "aligned")
    refused(nc, call(n_req=0), "requests")
    refused(nc, call(n_req=4097), "requests")
    refused(nc, call(max_new=-1), "requests")
    refused(nc, call(k=32), "x is not")
    refused(nc, call(x=nc.Tensor(16, None, nc.F32, 4, 64, 256)), "x is not")
    refused(nc, call(y=nc.Tensor(16, None, nc.F16, 4, 100, 208)), "base is not")
    refused(nc, call(y=nc.Tensor(16, None, nc.F32, 3, 100, 400)), "base is not")
    refused(nc, call(out=nc.Tensor(16, None, nc.F16, 4, 96, 192)), "out is not")
    refused(nc, call(out=nc.Tensor(16, None, nc.F16, 4, 100, 200)), "out is not")


def test_cache_bytes(nc):
    L, a, b = nc.lib(), C.c_size_t(), C.c_size_t()
    nc.check(L.nc_paged_cache_bytes(nc.F16, 100000, 64, 8, 128, C.byref(a), C.byref(b)))
    assert (a.value, b.value) == (100000 * 64 * 8 * 128 * 2, 0)
    nc.check(L.nc_paged_cache_bytes(nc.Q8, 3, 16, 5, 64, C.byref(a), C.byref(b)))
    assert (a.value, b.value) == (3 * 16 * 5 * 64, 3 * 16 * 5 * 2 * 2)
    refused(nc, L.nc_paged_cache_bytes(nc.Q4, 3, 16, 5, 64, C.byref(a), C.byref(b)), "dtype")


def test_nothing_to_do_is_no_error(nc):
    L = nc.lib()
    cache, batch, _ = structs(nc)
    batch.max_tokens = 0
    q = nc.Tensor(16, None, nc.F16, 0, 256, 512)
    kv = nc.Tensor(16, None, nc.F16, 0, 128, 256)
    assert L.nc_paged_attn(C.byref(q), C.byref(cache), C.byref(batch), C.byref(q), 4, 0, 0, None, 0, None) == 0
    assert L.nc_paged_append(C.byref(q), C.byref(kv), C.byref(kv), C.byref(q), C.byref(cache), C.byref(batch), None, 0, 0,
                             None) == 0


def test_results_over_inputs(nc):
    L = nc.lib()
    cache, batch, _ = structs(nc)
    at = 1 << 20
    row = lambda dtype, cols, data=at, pitch=0: nc.Tensor(data, None, dtype, 4, cols, pitch or  # noqa: E731
                                                          cols * (2 if dtype == nc.F16 else 4))
    q = row(nc.F16, 256)
    q8 = nc.Tensor(at, None, nc.Q8, 4, 256, 272)
    for out in (row(nc.F16, 256, at + 512), row(nc.F16, 256, at - 16), row(nc.F16, 256, at, 528), q8):
        refused(nc, L.nc_paged_attn(C.byref(q), C.byref(cache), C.byref(batch), C.byref(out), 4, 0, 0, None, 0, None),
                "lies over q")
    lora = nc.Lora(a=16, b=16, scale=16, n_adapters=3, rank=16, k=64, n=64)
    x, y = row(nc.F16, 64), row(nc.F32, 64, at << 1)

    def add(out, x=x, y=y):
        return L.nc_lora_add(C.byref(x), C.byref(y), C.byref(lora), 16, 16, 2, 2, C.byref(out), None)

    refused(nc, add(x), "over x")
    refused(nc, add(row(nc.F16, 64, at + 256)), "over x")
    refused(nc, add(row(nc.F32, 64, at - 512)), "over x")
    refused(nc, add(row(nc.F16, 64, at << 1)), "over base")
    refused(nc, add(row(nc.F32, 64, (at << 1) + 256)), "over base")
    refused(nc, add(row(nc.F32, 64, at << 1, 272)), "over base")


def test_workspace_follows_the_rows_that_can_use_it(nc):
    """One long chunk, or a few rows of it: not the rows of the chunk times the parts of a few."""
    L, size = nc.lib(), C.c_size_t()
    cache, batch, _ = structs(nc)
    cache.n_kv_heads, cache.d_head, cache.n_pages = 8, 128, 1 << 16
    batch.n_req, batch.max_tokens, batch.max_new, batch.max_kv, batch.max_pages = 1, 8192, 8192, 8192, 512
    nc.check(L.nc_paged_attn_workspace(C.byref(cache), C.byref(batch), 64, 0, 0, C.byref(size)))
    assert size.value < 64 << 20
    for n_req in (1, 64, 4096):
        for kv in (8192, 1 << 24):
            batch.n_req, batch.max_tokens, batch.max_new, batch.max_kv, batch.max_pages = n_req, n_req, 1, kv, kv // 16
            if n_req * batch.max_pages < 1 << 31:
                nc.check(L.nc_paged_attn_workspace(C.byref(cache), C.byref(batch), 64, 0, 0, C.byref(size)))
                assert size.value <= 1 << 30
