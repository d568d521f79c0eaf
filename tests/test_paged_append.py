"""nc_paged_append: the cache and the q rows hold what nc_rotary_emb and the row roundings give, and nothing else changes."""
import ctypes as C

import numpy as np
import pytest
import torch

import paged_util as P
from paged_util import Cache, Rows, Step, sync

pytestmark = pytest.mark.gpu


def rope_table(gpu, n, d, half):
    """(cos, sin) pairs; nc_rope_table's where its head size gives this many."""
    tab = np.zeros((n, max(half, 1), 2), np.float32)
    if half:
        gpu.check(gpu.lib().nc_rope_table(n, d, 2 * half / d, tab.ctypes.data_as(C.c_void_p)), "rope_table")
    return torch.from_numpy(tab[:, :half]).contiguous().cuda()


def append(gpu, s, cache, q, k, v, q_out, rope, half, rows=None, on=None):
    gpu.check(gpu.lib().nc_paged_append(q.ref if q else None, k.ref, v.ref, q_out.ref if q_out else None, cache.ref, s.ref,
                                        P.ptr(rope), (rope.shape[0] if rope is not None else 0) if rows is None else rows,
                                        half, on), "paged_append")


def turned(x, rope, pos):
    """fp32 rotation, in the order of nc_rotary_emb's operations, [n, heads, d]."""
    half = rope.shape[1]
    t = rope.cpu()[pos]
    c, s = t[:, None, :, 0], t[:, None, :, 1]
    lo, hi = x[..., :half], x[..., half:2 * half]
    return torch.cat([lo * c - hi * s, lo * s + hi * c, x[..., 2 * half:]], -1)


def snapshot(cache):
    return [t.clone() for t in (cache.k, cache.v, cache.kd, cache.vd) if t is not None]


CASES = [
    # (rows, q_out, cache, d, hq, hkv, page, half, new, past, pad)
    ("f16", "f16", "f16", 64, 4, 2, 16, 32, [1], [0], 0),
    ("f16", "f16", "f16", 64, 32, 4, 16, 32, [1, 1, 0, 1], [15, 16, 3, 700], 2),
    ("q8", "q8", "q8", 64, 6, 3, 16, 8, [5, 0, 33], [0, 9, 14], 3),
    ("f32", "q8", "q8", 64, 5, 5, 32, 32, [40, 7], [1, 60], 1),
    ("f32", "f16", "q8", 128, 3, 1, 64, 64, [9, 100], [63, 0], 0),
    ("q8", "f16", "f16", 128, 2, 2, 1024, 24, [3, 1030], [1020, 0], 0),
    ("f16", "q8", "f16", 128, 8, 8, 16, 0, [17], [3], 4),
    ("f32", "f16", "f16", 64, 2, 1, 16, 13, [20, 1], [0, 40], 0),  # pairs that are no multiple of 8
    ("q8", "q8", "q8", 128, 2, 1, 16, 61, [6], [11], 1),
    ("f16", "f16", "q8", 64, 2, 1, 16, 1, [6], [11], 1),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c[:8])))
def test_append(gpu, case):
    rows, qo, ckind, d, hq, hkv, page, half, new, past, pad = case
    g = torch.Generator().manual_seed(d + half)
    s = Step(new, past, page, g, pad=pad).planned()
    n, live = s.max_tokens, s.tokens
    x = [torch.randn(n, h * d, generator=g) * 3 for h in (hq, hkv, hkv)]
    q, k, v = (Rows(rows, n, t.shape[1], t, fill=0x7F) for t in x)
    out = Rows(qo, n, hq * d, fill=0x5A)
    cache = Cache(ckind, s.n_pages, page, hkv, d, fill=7.0)
    before, out_before = snapshot(cache), out.buf.clone()
    rope = rope_table(gpu, s.max_kv, d, half) if half else None
    append(gpu, s, cache, q, k, v, out, rope, half)
    sync()
    pos = torch.tensor(s.want_pos[:live])
    qv, kv, vv = (r.values().float().reshape(n, -1, d)[:live] for r in (q, k, v))
    if half:
        qv, kv = turned(qv, rope, pos), turned(kv, rope, pos)
    want_out = Rows(qo, n, hq * d, fill=0x5A)
    if live:
        stored = Rows(qo, live, hq * d, qv.reshape(live, -1), fill=0x5A)
        used = {"f16": hq * d * 2, "q8": hq * d // 32 * 34}[qo]
        want_out.buf[:live, :used] = stored.buf[:, :used]
    assert torch.equal(out.buf, want_out.buf), "q rows, or what lies beside them"
    want = Cache(ckind, s.n_pages, page, hkv, d, fill=7.0)
    want.put("k", s.want_slots[:live], kv)
    want.put("v", s.want_slots[:live], vv)
    for a, b in zip(snapshot(cache), snapshot(want)):
        assert torch.equal(a, b)
    assert len(before) == len(snapshot(want)) and torch.equal(out_before[live:], out.buf[live:])


@pytest.mark.parametrize("kind", ["f16", "q8"])
def test_same_as_rotary_emb(gpu, kind):
    """One request from position 0 in ascending pages: the cache's rows are nc_rotary_emb's, bit for bit."""
    L, n, heads, page = gpu.lib(), 50, 3, 16
    g = torch.Generator().manual_seed(9)
    s = Step([n], [0], page, g)
    s.want_table[0][:4] = [0, 1, 2, 3]
    s.want_slots = list(range(n))
    s.planned()
    k = Rows(kind, n, heads * 64, torch.randn(n, heads * 64, generator=g))
    rope = rope_table(gpu, n, 64, 32)
    turned_k = Rows(kind, n, heads * 64)
    gpu.check(L.nc_rotary_emb(k.ref, turned_k.ref, 64, 1.0, P.ptr(rope), 0, n, None), "rotary_emb")
    cache, q_out = Cache(kind, s.n_pages, page, heads, 64), Rows(kind, n, heads * 64)
    append(gpu, s, cache, k, k, k, q_out, rope, 32)
    sync()
    assert torch.equal(q_out.buf, turned_k.buf)
    assert torch.equal(cache.values("k", range(n)).reshape(n, -1), turned_k.values())
    assert torch.equal(cache.values("v", range(n)).reshape(n, -1), k.values())


@pytest.mark.parametrize("kind", ["f16", "q8"])
def test_q_in_place_and_absent(gpu, kind):
    g = torch.Generator().manual_seed(10)
    s = Step([7, 2], [3, 30], 16, g, pad=1).planned()
    x = [torch.randn(10, h * 64, generator=g) for h in (4, 2, 2)]
    rope = rope_table(gpu, s.max_kv, 64, 32)
    got = []
    for where in ("apart", "in place", "absent"):
        q, k, v = (Rows(kind, 10, t.shape[1], t) for t in x)
        out = {"apart": Rows(kind, 10, 256), "in place": q, "absent": None}[where]
        if where == "apart":
            out.buf[9:] = q.buf[9:]
        cache = Cache(kind, s.n_pages, 16, 2, 64)
        append(gpu, s, cache, q if out else None, k, v, out, rope, 32)
        sync()
        got.append((out.buf.clone() if out else None, snapshot(cache)))
    assert torch.equal(got[0][0], got[1][0])
    for other in got[1:]:
        assert all(torch.equal(a, b) for a, b in zip(got[0][1], other[1]))


def test_views_of_one_projection(gpu):
    """q, k and v as column ranges of one fp32 matrix, wider rows than their columns."""
    g = torch.Generator().manual_seed(11)
    hq, hkv, d, n = 4, 2, 64, 9
    s = Step([n], [2], 16, g).planned()
    x = torch.randn(n, (hq + 2 * hkv) * d, generator=g)
    whole = Rows("f32", n, (hq + 2 * hkv) * d, x)
    part = lambda at, h: gpu.Tensor(whole.buf.data_ptr() + 4 * at * d, None, gpu.F32, n, h * d, whole.pitch)  # noqa: E731
    q, k, v = part(0, hq), part(hq, hkv), part(hq + hkv, hkv)
    rope = rope_table(gpu, s.max_kv, d, 32)
    out, cache = Rows("f16", n, hq * d, extra_pitch=48), Cache("f16", s.n_pages, 16, hkv, d)
    gpu.check(gpu.lib().nc_paged_append(C.byref(q), C.byref(k), C.byref(v), out.ref, cache.ref, s.ref, P.ptr(rope),
                                        rope.shape[0], 32, None), "paged_append")
    sync()
    pos, heads = torch.tensor(s.want_pos), x.reshape(n, -1, d)
    assert torch.equal(out.values().half(), turned(heads[:, :hq], rope, pos).reshape(n, -1).half().double().half())
    assert torch.equal(cache.values("k", s.want_slots), turned(heads[:, hq:hq + hkv], rope, pos).half().double())
    assert torch.equal(cache.values("v", s.want_slots), heads[:, hq + hkv:].half().double())


def test_rows_outside_the_cache_or_the_table_are_passed_over(gpu):
    g = torch.Generator().manual_seed(12)
    s = Step([8], [0], 16, g).planned()
    s.slots.copy_(P.ints([-1, s.n_pages * 16, 3, 2 ** 31 - 1, -2 ** 31, 5, 6, 7]))
    s.positions.copy_(P.ints([0, 1, 4, 3, 4, -1, 2, 10 ** 9]))  # the table has rows 0 to 4
    x = torch.randn(8, 64, generator=g)
    rows = Rows("f16", 8, 64, x)
    out, cache = Rows("f16", 8, 64, fill=0x11), Cache("f16", s.n_pages, 16, 1, 64, fill=7.0)
    rope = rope_table(gpu, 5, 64, 32)
    append(gpu, s, cache, rows, rows, rows, out, rope, 32)
    sync()
    want = Cache("f16", s.n_pages, 16, 1, 64, fill=7.0)
    xs = x.half().float().reshape(8, 1, 64)[[2, 6]]
    want.put("k", [3, 6], turned(xs, rope, torch.tensor([4, 2])))
    want.put("v", [3, 6], xs)
    assert torch.equal(cache.k, want.k) and torch.equal(cache.v, want.v)
    touched = (out.buf != 0x11).any(1).nonzero().flatten().tolist()
    assert touched == [2, 6]


def test_values_without_a_finite_neighbour(gpu):
    """Zero rows, infinities and NaN: each value alone decides what is stored for it in fp16."""
    g = torch.Generator().manual_seed(13)
    s = Step([4], [0], 16, g).planned()
    x = torch.zeros(4, 64)
    x[1, 3], x[2, 5], x[3] = float("inf"), float("nan"), 70000.0
    rows = Rows("f32", 4, 64, x)
    cache = Cache("f16", s.n_pages, 16, 1, 64)
    append(gpu, s, cache, None, rows, rows, None, None, 0)
    sync()
    assert torch.equal(cache.values("v", s.want_slots).reshape(4, 64).nan_to_num(nan=-1.0),
                       x.half().double().nan_to_num(nan=-1.0))
    cache = Cache("q8", s.n_pages, 16, 1, 64, fill=3.0)
    zero = Rows("f32", 4, 64, torch.zeros(4, 64))
    append(gpu, s, cache, None, zero, zero, None, None, 0)
    sync()
    assert not cache.values("k", s.want_slots).any() and not cache.values("v", s.want_slots).any()
