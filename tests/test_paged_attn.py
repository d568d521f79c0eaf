"""nc_paged_attn against the softmax formula in 64 bits, within what its documented roundings can do to each value."""
import ctypes as C

import pytest
import torch

import paged_util as P
from paged_util import Cache, Rows, Step, attend, plain_attention, rounded, sync, within, workspace

pytestmark = pytest.mark.gpu


def make(new, past, page, d, hq, hkv, rows, ckind, seed=0, pad=0, fill=float("nan"), scale=1.0, **kw):
    """A planned step whose pages hold NaN wherever no position is cached."""
    g = torch.Generator().manual_seed(seed)
    s = Step(new, past, page, g, pad=pad, **kw).planned()
    cache = Cache(ckind, s.n_pages, page, hkv, d, fill=fill)
    for r in range(s.n_req):
        slots = s.past_slots(r)
        if slots:
            cache.put("k", slots, torch.randn(len(slots), hkv, d, generator=g) * scale)
            cache.put("v", slots, torch.randn(len(slots), hkv, d, generator=g))
    q = Rows(rows, s.max_tokens, hq * d, torch.randn(s.max_tokens, hq * d, generator=g) * scale)
    return s, cache, q


def check(s, cache, q, out, hq, window=0, sink=0, hidden=None, what=""):
    want, tol = plain_attention(s, cache, q, hq, window, sink, hidden)
    got = out.values()[:s.tokens]
    assert torch.isfinite(got).all(), what
    within(got, want, rounded(out.kind, want, tol), what)


CASES = {
    # name: (new, past, page, d, hq, hkv, rows, cache)
    "one token, nothing before it": ([1], [0], 16, 64, 4, 2, "f16", "f16"),
    "one token, 128 wide": ([1], [77], 16, 128, 8, 1, "f16", "f16"),
    "one kv head for 40": ([1, 3], [5, 200], 32, 64, 40, 1, "f16", "f16"),
    "ends of steps": ([1] * 9, [14, 15, 16, 30, 31, 32, 63, 126, 127], 16, 64, 4, 4, "f16", "f16"),
    "ends of steps, q8": ([1] * 9, [14, 15, 16, 30, 31, 32, 63, 126, 127], 16, 128, 4, 2, "q8", "q8"),
    "long enough to split": ([1, 1, 1], [3000, 5, 1500], 64, 64, 4, 1, "f16", "f16"),
    "long, q8": ([1, 1], [2500, 131], 128, 64, 3, 3, "f16", "q8"),
    "long, 128 wide, q8": ([1, 2], [1111, 1300], 16, 128, 4, 2, "f16", "q8"),
    "idle requests": ([0, 2, 0, 1], [30, 40, 0, 9], 16, 64, 6, 3, "f16", "f16"),
    "chunks": ([17, 1, 33, 5], [0, 90, 16, 31], 16, 64, 6, 2, "f16", "f16"),
    "chunks, q8": ([17, 1, 33, 5], [0, 90, 16, 31], 32, 64, 6, 2, "q8", "q8"),
    "chunks, q8 rows over fp16 pages": ([9, 20], [3, 50], 16, 128, 2, 2, "q8", "f16"),
    "a prompt from its start": ([130], [0], 16, 64, 2, 1, "f16", "f16"),
    "a prompt from its start, 128 wide": ([150], [0], 1024, 128, 3, 3, "f16", "q8"),
    "a long chunk over a long past": ([140, 1], [600, 1000], 64, 128, 8, 2, "f16", "f16"),
    "a long chunk, uneven group": ([90, 7], [100, 333], 16, 64, 6, 2, "q8", "q8"),
    "group that divides no tile": ([50], [20], 16, 64, 7, 1, "f16", "f16"),
}


@pytest.mark.parametrize("name", list(CASES))
def test_attention(gpu, name):
    new, past, page, d, hq, hkv, rows, ckind = CASES[name]
    s, cache, q = make(new, past, page, d, hq, hkv, rows, ckind, seed=len(name), pad=2)
    out = Rows(rows, s.max_tokens, hq * d, fill=0x3C)
    attend(s, cache, q, out, hq)
    sync()
    check(s, cache, q, out, hq, what=name)
    assert (out.buf[s.tokens:] == 0x3C).all()  # rows behind the last request


WINDOWS = [(1, 0), (1, 1), (16, 0), (16, 4), (31, 1), (33, 20), (100, 64), (1000, 4), (64, 5000), (2 ** 31 - 1, 2 ** 31 - 1)]


@pytest.mark.parametrize("window,sink", WINDOWS)
@pytest.mark.parametrize("shape", ["tokens", "chunks"])
def test_window_and_sinks(gpu, window, sink, shape):
    new, past = ([1, 1, 1, 1], [700, 0, 33, 95]) if shape == "tokens" else ([40, 3, 130], [300, 0, 17])
    for d, hq, hkv, rows, ckind, page in ((64, 4, 2, "f16", "f16", 16), (128, 2, 1, "f16", "q8", 32)):
        s, cache, q = make(new, past, page, d, hq, hkv, rows, ckind, seed=window % 1000 + sink % 1000)
        out = Rows(rows, s.max_tokens, hq * d)
        attend(s, cache, q, out, hq, window, sink)
        sync()
        check(s, cache, q, out, hq, window, sink, what=f"d={d}")


@pytest.mark.parametrize("ckind", ["f16", "q8"])
def test_pages_outside_the_window_may_be_gone(gpu, ckind):
    s, cache, q = make([1, 20], [500, 300], 16, 64, 4, 2, "f16", ckind, seed=3)
    window, sink = 50, 3
    want = Rows("f16", s.max_tokens, 256)
    attend(s, cache, q, want, 4, window, sink)
    for r in range(2):
        first = s.past[r] - window + 1  # of the first row
        for j in range(1, first // 16):
            s.table[r, j] = -1 if j % 2 else 2 ** 31 - 1
    out = Rows("f16", s.max_tokens, 256)
    attend(s, cache, q, out, 4, window, sink)
    sync()
    assert torch.equal(out.buf, want.buf)


@pytest.mark.parametrize("d,new,past", [(64, [1, 1], [60, 30]), (128, [1], [300]), (64, [40], [50]), (128, [200], [0])])
def test_entries_that_are_no_page_are_not_seen(gpu, d, new, past):
    s, cache, q = make(new, past, 16, d, 4, 2, "f16", "f16", seed=4)
    hidden = []
    for r in range(s.n_req):
        h = torch.zeros(s.new[r] + s.past[r], dtype=torch.bool)
        for j, bad in ((0, -1), (2, s.n_pages), (4, -2 ** 31)):
            if j < s.max_pages:
                s.table[r, j] = bad
                h[j * 16:(j + 1) * 16] = True
        hidden.append(h)
    out = Rows("f16", s.max_tokens, 4 * d)
    attend(s, cache, q, out, 4)
    sync()
    check(s, cache, q, out, 4, hidden=hidden)


def test_rows_that_see_nothing_are_zero(gpu):
    for new, past in (([1, 2], [0, 12]), ([1], [1500]), ([100], [30])):
        s, cache, q = make(new, past, 16, 64, 2, 1, "f16", "f16", seed=5)
        s.table.fill_(-1)
        out = Rows("f16", s.max_tokens, 128, fill=0x3C)
        attend(s, cache, q, out, 2)
        sync()
        assert not out.values().any()


@pytest.mark.parametrize("ckind", ["f16", "q8"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("new,past,hq,hkv", [([5], [20], 4, 2), ([3, 40], [33, 0], 2, 2), ([150], [40], 4, 1)])
def test_positions_to_come_have_no_effect(gpu, ckind, bad, new, past, hq, hkv):
    """A row whose k and v are not finite: rows before it are as if it were not there, rows that see it are not
    finite; through a window, rows past it are finite again."""
    d, window = 64, 24
    s, cache, q = make(new, past, 16, d, hq, hkv, "f16", ckind, seed=6)
    r, at = len(new) - 1, new[-1] // 2
    slot = [s.want_slots[s.want_rows[r] + at]]
    n_pages, _, page, _ = cache.shape
    if ckind == "f16":
        cache.k[slot[0] // page, :, slot[0] % page] = bad
        cache.v[slot[0] // page, :, slot[0] % page] = bad
    else:
        cache.kd[slot[0] // page, :, slot[0] % page] = bad
        cache.vd[slot[0] // page, :, slot[0] % page] = bad
    for win in (0, window):
        out = Rows("f16", s.max_tokens, hq * d)
        attend(s, cache, q, out, hq, win, 0)
        sync()
        got = out.values()
        i = torch.arange(s.tokens) - s.want_rows[r]
        sees = (i >= at) & ((i < at + win) if win else True)
        assert torch.isfinite(got[~sees]).all()
        assert not torch.isfinite(got[sees]).any(1).any() or bad == float("inf")
        assert not torch.isfinite(got[sees]).all(1).any()
        clean = Cache(ckind, *[cache.shape[j] for j in (0, 2, 1, 3)])
        for name in ("k", "v", "kd", "vd"):
            if getattr(cache, name) is not None:
                getattr(clean, name).copy_(getattr(cache, name))
        clean.put("k", slot, torch.zeros(1, hkv, d))
        clean.put("v", slot, torch.zeros(1, hkv, d))
        want = Rows("f16", s.max_tokens, hq * d)
        attend(s, clean, q, want, hq, win, 0)
        sync()
        assert torch.equal(got[~sees], want.values()[~sees])


def test_large_scores(gpu):
    """Scores of some hundreds: one weight near 1, the others vanish; and equal scores everywhere."""
    for scale in (12.0, 0.0):
        for new, past in (([1], [900]), ([70], [10])):
            s, cache, q = make(new, past, 16, 64, 4, 2, "f16", "f16", seed=7, scale=scale)
            out = Rows("f16", s.max_tokens, 256)
            attend(s, cache, q, out, 4)
            sync()
            check(s, cache, q, out, 4, what=f"scale {scale}")


@pytest.mark.parametrize("new,past", [([1], [9000]), ([80], [9000])])
def test_many_small_weights(gpu, new, past):
    """One weight of 1 and thousands of 2^-25: what is below fp16's smallest number still counts."""
    s, cache, q = make(new, past, 64, 64, 1, 1, "f16", "f16", seed=8)
    n = past[0] + new[0]
    k, v = torch.zeros(n, 1, 64), torch.ones(n, 1, 64)
    k[0, 0, 0], v[0] = 25 * 0.6931471805599453 * 8 / 16, 0.0
    cache.put("k", s.past_slots(0), k)
    cache.put("v", s.past_slots(0), v)
    x = torch.zeros(new[0], 64)
    x[:, 0] = 16.0
    q = Rows("f16", new[0], 64, x)
    out = Rows("f16", new[0], 64)
    attend(s, cache, q, out, 1)
    sync()
    want, tol = plain_attention(s, cache, q, 1)
    assert 2e-4 < want.min() and want.max() < 3e-4
    within(out.values(), want, rounded("f16", want, want * 2.0 ** -9), "small weights")


def test_same_results_every_time_and_on_another_stream(gpu):
    for new, past in (([1, 1, 1], [2000, 900, 17]), ([150, 1], [700, 2000])):
        s, cache, q = make(new, past, 16, 64, 8, 2, "f16", "f16", seed=9)
        first = Rows("f16", s.max_tokens, 512)
        attend(s, cache, q, first, 8)
        sync()
        streams = [torch.cuda.Stream() for _ in range(3)]
        outs = [Rows("f16", s.max_tokens, 512) for _ in streams]
        works = [workspace(s, cache, 8, 0, 0) for _ in streams]  # calls that overlap have their own
        sync()
        for _ in range(4):
            for st, out, work in zip(streams, outs, works):
                attend(s, cache, q, out, 8, work=work, on=P.stream(st))
        sync()
        for out in outs:
            assert torch.equal(out.buf, first.buf)


def test_two_captured_graphs_replayed(gpu):
    """Lengths change between replays, within the bounds that the capture was made with."""
    hq, hkv, d = 4, 2, 64
    s, cache, q = make([3, 1, 6], [900, 40, 100], 16, d, hq, hkv, "f16", "f16", seed=10, max_kv=1200, max_new=8)
    graphs = []
    for window in (0, 64):
        out, work = Rows("f16", s.max_tokens, hq * d), workspace(s, cache, hq, window, 2)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
            attend(s, cache, q, out, hq, window, 2, work, P.stream(torch.cuda.current_stream()))
        graphs.append((window, graph, out, work))
    for kv in ([903, 41, 106], [30, 9, 6], [500, 41, 7], [903, 1, 106]):
        s.kv_len.copy_(P.ints(kv))
        for window, graph, out, _ in graphs:
            out.buf.zero_()
            graph.replay()
            sync()
            eager = Rows("f16", s.max_tokens, hq * d)
            attend(s, cache, q, eager, hq, window, 2)
            sync()
            assert torch.equal(out.buf, eager.buf), (kv, window)
            s.past = [k - n for k, n in zip(kv, s.new)]
            check(s, cache, q, out, hq, window, 2, what=str(kv))


def test_lengths_beyond_the_bounds_leave_rows_alone(gpu):
    s, cache, q = make([2, 3, 1], [20, 10, 5], 16, 64, 2, 1, "f16", "f16", seed=11)
    good = Rows("f16", s.max_tokens, 128, fill=0x3C)
    attend(s, cache, q, good, 2)
    for kv, rows in (([2 ** 31 - 1, 13, 6], range(0, 2)), ([22, -1, 6], range(2, 5)), ([22, 13, 0], range(5, 6))):
        s.kv_len.copy_(P.ints(kv))
        out = Rows("f16", s.max_tokens, 128, fill=0x3C)
        attend(s, cache, q, out, 2)
        sync()
        for i in range(6):
            assert (out.buf[i] == 0x3C).all() if i in rows else torch.equal(out.buf[i], good.buf[i]), (kv, i)


def test_row_starts_that_lead_nowhere(gpu):
    """Tables of garbage: rows outside the tensors are not touched, and the call ends."""
    s, cache, q = make([2, 3, 1], [20, 10, 5], 16, 64, 2, 1, "f16", "f16", seed=12, pad=3)
    big = 2 ** 31 - 1
    for starts in ([0, -5, 4, 6], [big, big, big, big], [-big, big, 0, 3], [6, 5, 2, 0], [0, 9, 9, 10 ** 6]):
        s.row_start.copy_(P.ints(starts))
        whole = torch.full((s.max_tokens + 8, 256), 0x3C, dtype=torch.uint8, device="cuda")
        t = gpu.Tensor(whole[4:].data_ptr(), None, gpu.F16, s.max_tokens, 128, 256)
        work = workspace(s, cache, 2, 0, 0)
        gpu.check(gpu.lib().nc_paged_attn(q.ref, cache.ref, s.ref, C.byref(t), 2, 0, 0, P.ptr(work[0]), work[1], None))
        sync()
        assert (whole[:4] == 0x3C).all() and (whole[4 + s.max_tokens:] == 0x3C).all(), starts


def test_pages_past_32_bit_offsets(gpu):
    """Pages whose bytes lie beyond 4 GiB of the cache, and values beyond 2^31."""
    page, hkv, d = 64, 8, 128
    first = (1 << 32) // (page * hkv * d) + 3  # values past 2^32
    g = torch.Generator().manual_seed(13)
    for new, past in (([1, 1], [300, 40]), ([70], [100])):
        s = Step(new, past, page, g, first_page=first).planned()
        cache = Cache("f16", 1, page, hkv, d)
        cache.k, cache.v = (torch.empty(s.n_pages, hkv, page, d, dtype=torch.float16, device="cuda") for _ in range(2))
        cache.shape = tuple(cache.k.shape)
        cache.t.k, cache.t.v, cache.t.n_pages = P.ptr(cache.k), P.ptr(cache.v), s.n_pages
        for r in range(s.n_req):
            slots = s.past_slots(r)
            cache.put("k", slots, torch.randn(len(slots), hkv, d, generator=g))
            cache.put("v", slots, torch.randn(len(slots), hkv, d, generator=g))
        x = torch.randn(s.tokens, 8 * d, generator=g)
        rows, out = Rows("f16", s.tokens, 8 * d, x), Rows("f16", s.tokens, 8 * d)
        k, v = (Rows("f16", s.tokens, hkv * d, torch.randn(s.tokens, hkv * d, generator=g)) for _ in range(2))
        gpu.check(gpu.lib().nc_paged_append(None, k.ref, v.ref, None, cache.ref, s.ref, None, 0, 0, None))
        attend(s, cache, rows, out, 8)
        sync()
        live = s.want_slots[:s.tokens]
        assert torch.equal(cache.values("k", live).reshape(s.tokens, -1), k.values())
        check(s, cache, rows, out, 8)
        del cache
        torch.cuda.empty_cache()


def test_q8_rows_out_of_fp16_rows(gpu):
    """The result's type is its own choice."""
    for new, past in (([1, 1], [100, 2]), ([40], [30])):
        s, cache, q = make(new, past, 16, 64, 4, 2, "f16", "q8", seed=14)
        out = Rows("q8", s.max_tokens, 256)
        attend(s, cache, q, out, 4)
        sync()
        check(s, cache, q, out, 4)


def test_wider_pitches(gpu):
    s, cache, _ = make([3, 40], [20, 0], 16, 64, 4, 2, "f16", "f16", seed=15)
    x = torch.randn(s.max_tokens, 256, generator=torch.Generator().manual_seed(1))
    tight, wide = Rows("f16", s.max_tokens, 256, x), Rows("f16", s.max_tokens, 256, x, fill=0x7F, extra_pitch=80)
    a, b = Rows("f16", s.max_tokens, 256), Rows("f16", s.max_tokens, 256, fill=0x3C, extra_pitch=16)
    attend(s, cache, tight, a, 4)
    attend(s, cache, wide, b, 4)
    sync()
    assert torch.equal(a.values(), b.values()) and (b.buf[:, 512:] == 0x3C).all()


@pytest.mark.parametrize("d,ckind", [(64, "f16"), (128, "q8")])
def test_chunks_over_more_positions_than_one_lookup_holds(gpu, d, ckind):
    """128-row tiles look 16384 positions' pages up at a time; entries in the second lot that are no page, too."""
    s, cache, q = make([60, 3], [20000, 17000], 64, d, 2, 1, "f16", ckind, seed=16)
    out = Rows("f16", s.max_tokens, 2 * d)
    attend(s, cache, q, out, 2)
    sync()
    check(s, cache, q, out, 2)
    hidden = [torch.zeros(s.new[r] + s.past[r], dtype=torch.bool) for r in range(2)]
    for r in range(2):
        for j in (3, 259, 260):
            s.table[r, j] = -1
            hidden[r][j * 64:(j + 1) * 64] = True
    attend(s, cache, q, out, 2)
    sync()
    check(s, cache, q, out, 2, hidden=hidden)


@pytest.mark.parametrize("n_req", [65, 150, 700])
def test_many_requests(gpu, n_req):
    """Single tokens, chunks and idle requests side by side, more than one probe of a wavefront finds."""
    g = torch.Generator().manual_seed(n_req)
    new = (torch.randint(0, 70, (n_req,), generator=g) * (torch.rand(n_req, generator=g) < 0.3)).tolist()
    new = [n if n or i % 3 else 1 for i, n in enumerate(new)]
    past = torch.randint(0, 40, (n_req,), generator=g).tolist()
    for hq, hkv, rows in ((2, 1, "f16"), (1, 1, "q8")):
        s, cache, q = make(new, past, 16, 64, hq, hkv, rows, rows, seed=n_req)
        out = Rows(rows, s.max_tokens, hq * 64)
        attend(s, cache, q, out, hq)
        sync()
        check(s, cache, q, out, hq)


@pytest.mark.parametrize("rows,ckind", [("f16", "f16"), ("q8", "q8"), ("f16", "q8")])
def test_q_in_place(gpu, rows, ckind):
    """out may be q: every kind of tile, joined parts among them, reads a row's head before it writes it."""
    s, cache, q = make([1, 0, 3, 40, 150], [5000, 4, 700, 64, 300], 32, 64, 4, 2, rows, ckind, seed=18, pad=2)
    out = Rows(rows, s.max_tokens, 256)
    attend(s, cache, q, out, 4)
    attend(s, cache, q, q, 4)
    sync()
    assert torch.equal(q.buf[:s.tokens], out.buf[:s.tokens])


@pytest.mark.parametrize("new,past", [([1, 1, 1], [100, 3000, 0]), ([1, 20, 0, 130], [900, 5, 70, 2000])])
@pytest.mark.parametrize("d,ckind", [(64, "q8"), (128, "f16")])
def test_looser_bounds(gpu, new, past, d, ckind):
    """Bounds far above the lengths: parts and tiles that hold nothing, other shapes of the launch."""
    for max_new, max_kv in ((200, 2200), (1000, 70000), (200, 1 << 20)):
        s, cache, q = make(new, past, 32, d, 4, 2, "f16", ckind, seed=19, max_new=max_new, max_kv=max(max_kv, 3001))
        out = Rows("f16", s.max_tokens, 4 * d)
        attend(s, cache, q, out, 4)
        sync()
        check(s, cache, q, out, 4)
