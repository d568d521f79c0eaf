"""The operators of batched serving, as cases that can be timed.

A server that runs many requests at once over one set of weights keeps every
request's K/V rows in pages of a common cache.  Each step it

  plan     turns the requests' lengths into block tables, slots and positions
           (nc_paged_plan)
  lora     adds each request's low-rank adapter to a shared projection
           (nc_lora_add)
  append   rotates the step's q and k rows at their own positions and stores
           k and v in the cache's slots (nc_paged_append)
  attn     attends from each request's new rows to its pages, single tokens
           and chunks of a prompt alike, over everything before them or over
           a window and the first few tokens (nc_paged_attn)

`run` computes these in their plain form (elementary torch operations in 32
bits), or with `own` set through the library.  Rows, caches and tables are
torch tensors in the library's layouts; Q8 rows and caches come back as the
values that they stand for.
"""
import ctypes as C
import importlib.util
import math
import os
import random
import sys

import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def listed():
    return [
        # the smallest step of a chat server: a few requests, one token each
        dict(name="plan-8", op="plan", n_req=8, lo=1, hi=1, past=1000, page=16, pad=0),
        # a large step of ragged prompt chunks and single tokens, some requests idle
        dict(name="plan-500", op="plan", n_req=500, lo=0, hi=250, past=4000, page=16, pad=37),
        # one token of seventeen requests in a small grouped-head fp16 model
        dict(name="append-f16-17", op="append", n_req=17, lo=1, hi=1, past=700, hq=32, hkv=4, d=64, rope=1.0, page=16,
             rows="f16", out="f16", pad=0),
        # prompt chunks of a Q8 model: raw fp32 projections to Q8 q rows and an 8-bit cache
        dict(name="append-q8-2000", op="append", n_req=3, lo=500, hi=900, past=1200, hq=36, hkv=36, d=64, rope=1.0,
             page=16, rows="f32", out="q8", pad=5),
        # one chat, one token, some way into the reply: latency
        dict(name="attn-f16-1", op="attn", n_req=1, lo=1, hi=1, past=700, hq=32, hkv=4, d=64, page=16, rows="f16",
             cache="f16", window=0, sink=0, pad=0),
        # a full decode batch with long, ragged contexts: the K/V bytes
        dict(name="attn-f16-64", op="attn", n_req=64, lo=1, hi=1, past=8000, hq=32, hkv=8, d=128, page=64, rows="f16",
             cache="f16", window=0, sink=0, pad=0),
        # a decode batch over an 8-bit cache, as many kv heads as heads
        dict(name="attn-q8-40", op="attn", n_req=40, lo=1, hi=1, past=3900, hq=36, hkv=36, d=64, page=16, rows="f16",
             cache="q8", window=0, sink=0, pad=0),
        # chunks of several long prompts over what is cached of them
        dict(name="attn-f16-chunk", op="attn", n_req=4, lo=500, hi=520, past=2000, hq=32, hkv=4, d=64, page=16,
             rows="f16", cache="f16", window=0, sink=0, pad=3),
        # long documents under a sliding window with a few sinks
        dict(name="attn-f16-window", op="attn", n_req=2, lo=900, hi=1100, past=11000, hq=32, hkv=8, d=128, page=64,
             rows="f16", cache="f16", window=1024, sink=4, pad=0),
        # a mixed step of a Q8 model: one prompt's chunk among single tokens
        dict(name="attn-q8-mixed", op="attn", n_req=12, lo=1, hi=400, past=3000, hq=32, hkv=32, d=64, page=32,
             rows="q8", cache="q8", window=0, sink=0, pad=1),
        # one token each of many requests with their own adapters, q|k|v of a grouped-head model
        dict(name="lora-f16-32", op="lora", n_req=32, lo=1, hi=1, adapters=24, rank=16, k=2048, n=2560, rows="f16",
             out="f16", pad=0),
        # prompt chunks under a few adapters of a higher rank, a wide projection's raw fp32 rows
        dict(name="lora-q8-chunk", op="lora", n_req=9, lo=40, hi=300, adapters=5, rank=64, k=2304, n=5760, rows="q8",
             out="f32", pad=2),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(c):
    w = work(c)
    return max(w["bytes"], w["flops"] / 50)


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        op = rng.choice(["plan", "append", "attn", "attn", "attn", "attn", "lora", "lora"])
        c = dict(op=op, n_req=_log_int(rng, 1, 500 if op == "plan" else 64))
        how = rng.random()  # single tokens, chunks, or both in one step
        hi = 1 if how < 0.4 else _log_int(rng, 2, 1000)
        c.update(lo=1 if how < 0.4 else rng.choice([0, 1, max(1, hi // 2)]), hi=hi, pad=rng.choice([0, 0, 1, 30]))
        if op != "lora":
            c.update(past=_log_int(rng, 1, 8000), page=rng.choice([16, 32, 64, 128]))
        if op in ("append", "attn"):
            hq, hkv, d = rng.choice([(32, 4, 64), (36, 36, 64), (32, 32, 64), (16, 4, 64), (20, 5, 64), (24, 6, 64),
                                     (12, 3, 64), (32, 8, 128), (16, 2, 128), (8, 8, 128)])
            c.update(hq=hq, hkv=hkv, d=d)
        if op == "append":
            c.update(rope=rng.choice([1.0, 0.25]), rows=rng.choice(["f16", "q8", "f32"]), out=rng.choice(["f16", "q8"]))
        elif op == "attn":
            rows = rng.choice(["f16", "q8"])
            c.update(rows=rows, cache="q8" if rows == "q8" else rng.choice(["f16", "f16", "q8"]))
            window = rng.choice([0, 0, _log_int(rng, 16, 2048)])
            c.update(window=window, sink=rng.choice([0, 1, 4, 20]) if window else 0)
        elif op == "lora":
            c.update(adapters=rng.randint(1, 24), rank=rng.choice([4, 8, 16, 24, 32, 64, 100, 128]),
                     k=rng.choice([1280, 1536, 2048, 2304, 5632]), n=rng.choice([768, 1000, 2048, 2560, 5760, 7168]),
                     rows=rng.choice(["f16", "q8"]), out=rng.choice(["f16", "q8", "f32"]))
        new, past = _lengths(c)
        tokens = sum(new)
        if not tokens or tokens > 40000 or (op == "append" and tokens > 4000) or (op == "lora" and tokens > 3000):
            continue
        # the plain form's padded scores and gathered pages
        if op == "attn" and len(new) * max(n + p for n, p in zip(new, past)) * max(
                max(new) * c["hq"], 2 * c["hkv"] * c["d"]) > 1 << 30:
            continue
        if _cost(c) <= most:
            return c


# ---- inputs ------------------------------------------------------------------


def _lengths(c):
    """New and cached rows of each request: the case's own, whatever the seed."""
    rng = random.Random(7919 * c["n_req"] + 31 * c["hi"] + c.get("past", 0))

    new, past = [], []
    for r in range(c["n_req"]):
        u, v = rng.random(), rng.random()
        # chunked steps are mostly single tokens with some long chunks where lo is 1
        n = c["lo"] + int((c["hi"] - c["lo"] + 1) * (u ** 6 if c["lo"] == 1 else u))
        new.append(min(n, c["hi"]))
        past.append(int(c.get("past", 0) * (0.02 + 0.98 * v)))
    new[c["n_req"] // 2], past[0] = c["hi"], c.get("past", 0)  # the longest of each
    return new, past


class _State:
    pass


def _up(a, b):
    return (a + b - 1) // b


def _q8_pitch(cols):
    return (cols // 32 * 34 + 15) // 16 * 16


def _block_codes(x):
    """Q8 codes and fp16 deltas of 32-value blocks along the last axis."""
    b = x.reshape(*x.shape[:-1], -1, 32)
    delta = b.abs().amax(-1, keepdim=True) / 127
    q = b * torch.where(delta > 0, 1 / delta, torch.zeros_like(delta))
    q = torch.sign(q) * torch.floor(q.abs().double() + 0.5).float()
    return q.reshape(x.shape), delta[..., 0].half()


def _values(codes, deltas):
    """The fp32 values of Q8 codes and their blocks' deltas."""
    c = codes.float().reshape(*codes.shape[:-1], -1, 32)
    return (c * deltas.float()[..., None]).reshape(codes.shape)


def _make_rows(kind, x):
    """Rows of values in the library's layout of a dtype."""
    if kind != "q8":
        return x.half() if kind == "f16" else x.float()
    n, cols = x.shape
    q, delta = _block_codes(x)
    buf = torch.zeros(n, _q8_pitch(cols), dtype=torch.uint8, device="cuda")
    buf[:, :cols] = q.to(torch.int8).view(torch.uint8)
    buf[:, cols:cols // 32 * 34] = delta.contiguous().view(torch.uint8)
    return buf


def _read_rows(kind, buf, cols):
    """The fp32 values of rows in the library's layout."""
    if kind != "q8":
        return buf.float()
    return _values(buf[:, :cols].view(torch.int8), buf[:, cols:cols // 32 * 34].view(torch.float16))


def _empty_rows(kind, n, cols):
    if kind == "q8":
        return torch.zeros(n, _q8_pitch(cols), dtype=torch.uint8, device="cuda")
    return torch.zeros(n, cols, dtype=torch.float16 if kind == "f16" else torch.float32, device="cuda")


def _round_rows(kind, x):
    """What rows of a dtype hold of fp32 values (Q8: as fp16 values)."""
    if kind != "q8":
        return x.half() if kind == "f16" else x
    pad = -x.shape[1] % 32
    q, delta = _block_codes(torch.nn.functional.pad(x, (0, pad)))
    return _values(q, delta)[:, :x.shape[1]].half()


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _random(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def _pages(c, s, g):
    """Lengths, a page pool in random order and the requests' block tables."""
    new, past = _lengths(c)
    page = c["page"]
    s.tokens = sum(new)
    s.max_tokens, s.max_new, s.max_kv = s.tokens + c["pad"], max(new), max(n + p for n, p in zip(new, past))
    s.max_pages = _up(s.max_kv, page) + 1
    have = [_up(p, page) for p in past]
    add = [_up(p + n, page) - h for n, p, h in zip(new, past, have)]
    s.n_pages = sum(have) + sum(add) + 9
    order = torch.randperm(s.n_pages, generator=g, device="cuda").to(torch.int32)
    s.new_len, s.seq_len = _ints(new), _ints(past)
    at = torch.arange(s.max_pages, device="cuda")[None]
    first = _ints([sum(have[:r]) for r in range(len(have))])[:, None]
    s.table = torch.where(at < _ints(have)[:, None], order[(first + at).clamp(max=s.n_pages - 1)], -1).to(torch.int32)
    s.n_free = s.n_pages - sum(have)
    s.free_pages = torch.zeros(s.n_pages, dtype=torch.int32, device="cuda")
    s.free_pages[:s.n_free] = order[sum(have):]
    s.pool = _ints([s.n_free, 0, 0, 0])


def prepare(case, seed):
    c, g = case, _random(seed)
    s = _State()
    s.case, s.seed = c, seed
    if c["op"] == "lora":
        _prepare_lora(c, s, g)
        return s
    _pages(c, s, g)
    n, page = s.max_tokens, c["page"]
    if c["op"] == "plan":
        s.row_start, s.kv_len = _ints([0] * (c["n_req"] + 1)), _ints([0] * c["n_req"])
        s.positions, s.slots = _ints([0] * n), _ints([0] * n)
        return s
    # the plan of this step
    s.row_start, s.kv_len, s.positions, s.slots, s.table, s.pool = _plan(s)
    s.table = s.table.contiguous()
    hq, hkv, d = c["hq"], c["hkv"], c["d"]
    shape = (s.n_pages, hkv, page, d)
    if c["op"] == "append":
        s.q, s.k, s.v = (_make_rows(c["rows"], _normal(g, n, h * d)) for h in (hq, hkv, hkv))
        half = int(d * c["rope"]) // 2
        angle = torch.arange(s.max_kv, device="cuda").double()[:, None] * 10000.0 ** (
            -torch.arange(half, device="cuda").double() / half)
        s.rope = torch.stack([angle.cos(), angle.sin()], -1).float().contiguous()
        s.q_out = _empty_rows(c["out"], n, hq * d)
        cache = c["out"]
    else:
        # q and k as a trained model's: channels of unequal size
        gain = torch.exp(0.3 * _normal(g, hkv, 1, d))
        s.q = _make_rows(c["rows"], (_normal(g, n, hkv, hq // hkv, d) * 1.5 / gain.permute(1, 0, 2)[:, :, None]).reshape(
            n, hq * d))
        s.out = _empty_rows(c["rows"], n, hq * d)
        cache = c["cache"]
    s.cache = cache
    if cache == "f16":
        s.kc, s.vc = (torch.zeros(shape, dtype=torch.float16, device="cuda") for _ in range(2))
        s.kd = s.vd = None
    else:
        s.kc, s.vc = (torch.zeros(shape, dtype=torch.int8, device="cuda") for _ in range(2))
        s.kd, s.vd = (torch.zeros(*shape[:3], d // 32, dtype=torch.float16, device="cuda") for _ in range(2))
    if c["op"] == "attn":
        step = max(1, (1 << 26) // (hkv * page * d))  # pages at a time
        for a in range(0, s.n_pages, step):
            b = min(s.n_pages, a + step)
            k, v = _normal(g, b - a, *shape[1:]) * gain, _normal(g, b - a, *shape[1:])
            if cache == "f16":
                s.kc[a:b], s.vc[a:b] = k.half(), v.half()
            else:
                for x, codes, deltas in ((k, s.kc, s.kd), (v, s.vc, s.vd)):
                    q, delta = _block_codes(x)
                    codes[a:b], deltas[a:b] = q.to(torch.int8), delta
    return s


def _prepare_lora(c, s, g):
    new, _ = _lengths(c)
    s.tokens = sum(new)
    s.max_tokens, s.max_new = s.tokens + c["pad"], max(new)
    s.row_start = _ints([sum(new[:r]) for r in range(len(new) + 1)])
    # adapter -1: a request of the model itself
    s.adapter = torch.randint(-1, c["adapters"], (c["n_req"],), generator=g, device="cuda").to(torch.int32)
    s.x = _make_rows(c["rows"], _normal(g, s.max_tokens, c["k"]))
    s.a = (_normal(g, c["adapters"], c["rank"], c["k"]) * c["k"] ** -0.5).half()
    s.b = (_normal(g, c["adapters"], c["n"], c["rank"]) * 0.3).half()
    s.scale = torch.rand(c["adapters"], generator=g, device="cuda") * 2 / c["rank"] ** 0.5
    s.base = _normal(g, s.max_tokens, c["n"])
    s.out = _empty_rows(c["out"], s.max_tokens, c["n"]) if c["out"] != "q8" else torch.zeros(
        s.max_tokens, (_up(c["n"], 32) * 34 + 15) // 16 * 16, dtype=torch.uint8, device="cuda")


# ---- one pass: the plain forms -------------------------------------------------


def _row_requests(row_start, n):
    """The request of each of n rows (the last one's for rows past the end) and whether it has one."""
    t = torch.arange(n, device="cuda")
    r = torch.searchsorted(row_start[1:].contiguous().long(), t, right=True)
    return t, r.clamp(max=row_start.shape[0] - 2), t < row_start[-1]


def _plan(s):
    page, n = s.case["page"], s.max_tokens
    new, seq, free = s.new_len.long(), s.seq_len.long(), s.free_pages.long()
    kv = seq + new
    have, need = (seq + page - 1) // page, (kv + page - 1) // page
    add = need - have
    before = torch.cumsum(add, 0) - add
    row_start = torch.nn.functional.pad(torch.cumsum(new, 0), (1, 0))
    n_free = s.pool[0].long()
    bad = ((new < 0) | (new > s.max_new)).any().long() * 8 + (row_start[-1] > n).long() * 4
    bad = bad + (need > s.max_pages).any().long() * 2 + (add.sum() > n_free).long()
    ok = bad == 0
    at = torch.arange(s.max_pages, device="cuda")[None]
    fresh = n_free - 1 - before[:, None] + have[:, None] - at
    table = torch.where(ok & (at >= have[:, None]) & (at < need[:, None]),
                        free[fresh.clamp(0, free.shape[0] - 1)], s.table.long())
    t, r, live = _row_requests(row_start, n)
    live = live & ok
    pos = seq[r] + t - row_start[r]
    slot = table[r, (pos // page).clamp(0, s.max_pages - 1)] * page + pos % page
    pool = torch.stack([n_free, n_free - torch.where(ok, add.sum(), 0), bad, torch.zeros_like(bad)])
    out = (torch.where(ok, row_start, 0), torch.where(ok, kv, seq), torch.where(live, pos, -1),
           torch.where(live, slot, -1), table, pool)
    return tuple(v.to(torch.int32) for v in out)


def _rotate(x, rope):
    half = rope.shape[1]
    cos, sin = rope[:, None, :, 0], rope[:, None, :, 1]
    lo, hi = x[..., :half], x[..., half:2 * half]
    return torch.cat([lo * cos - hi * sin, lo * sin + hi * cos, x[..., 2 * half:]], -1)


def _append(s):
    c = s.case
    n, d, page = s.max_tokens, c["d"], c["page"]
    live = s.slots[:s.tokens].long()  # the rows behind the last request stay as they were
    rope = s.rope[s.positions[:s.tokens].long()]
    q, k, v = (_read_rows(c["rows"], x, h * d)[:s.tokens].reshape(s.tokens, h, d)
               for x, h in ((s.q, c["hq"]), (s.k, c["hkv"]), (s.v, c["hkv"])))
    q, k = _rotate(q, rope), _rotate(k, rope)
    at = (live // page, slice(None), live % page)
    pad = torch.nn.functional.pad(q.reshape(s.tokens, -1), (0, 0, 0, n - s.tokens))
    if c["out"] == "f16":
        s.kc[at], s.vc[at] = k.half(), v.half()
        return pad.half(), s.kc, s.vc
    return (_round_rows("q8", pad),) + tuple(
        _round_rows("q8", x.reshape(s.tokens, -1)).reshape(s.tokens, -1, d) for x in (k, v))


def _gather(codes, deltas, pages):
    """fp32 [request, kv head, position, d] of the requests' pages."""
    x = codes[pages].float() if deltas is None else _values(codes[pages], deltas[pages])
    x = x.permute(0, 2, 1, 3, 4)
    return x.reshape(x.shape[0], x.shape[1], -1, x.shape[-1])


def _attn(s):
    c = s.case
    n, hq, hkv, d, page = s.max_tokens, c["hq"], c["hkv"], c["d"], c["page"]
    group, n_req = hq // hkv, c["n_req"]
    pages = s.table[:, :_up(s.max_kv, page)].long().clamp(min=0)
    kv, first, new = s.kv_len.long(), s.row_start[:-1].long(), s.new_len.long()
    k, v = _gather(s.kc, s.kd, pages), _gather(s.vc, s.vd, pages)
    key = torch.arange(k.shape[2], device="cuda")
    v = torch.where((key < kv[:, None])[:, None, :, None], v, 0)  # nothing of the pages' unused ends
    i = torch.arange(s.max_new, device="cuda")
    q = _read_rows(c["rows"], s.q, hq * d)[(first[:, None] + i).clamp(max=n - 1)]
    q = q.reshape(n_req, s.max_new, hkv, group, d).permute(0, 2, 3, 1, 4).reshape(n_req, hkv, group * s.max_new, d)
    score = torch.matmul(q, k.transpose(2, 3).contiguous()) * (1 / math.sqrt(d))
    pos = (kv - new)[:, None] + i
    seen = (key <= pos[..., None]) & (key < kv[:, None, None])
    if c["window"]:
        seen = seen & ((key > pos[..., None] - c["window"]) | (key < c["sink"]))
    score = score.reshape(n_req, hkv, group, s.max_new, -1).masked_fill(~seen[:, None, None], -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.reshape(n_req, hkv, group * s.max_new, -1), v).reshape(n_req, hkv, group, s.max_new, d)
    out = torch.where(total > 0, out / total, 0).permute(0, 3, 1, 2, 4).reshape(n_req, s.max_new, hq * d)
    t, r, live = _row_requests(s.row_start, n)
    out = torch.where(live[:, None], out[r, (t - first[r]).clamp(0, s.max_new - 1)], 0)
    return _round_rows(c["rows"], out)


def _lora(s):
    c = s.case
    n, count, rank = s.max_tokens, c["adapters"], c["rank"]
    _, r, live = _row_requests(s.row_start, n)
    mine = torch.where(live, s.adapter.long()[r], -1)
    x = _read_rows(c["rows"], s.x, c["k"])
    # every adapter's product, each row keeping its own adapter's
    t = torch.matmul(x, s.a.float().reshape(count * rank, c["k"]).T.contiguous()).reshape(n, count, rank)
    t = torch.where((torch.arange(count, device="cuda") == mine[:, None])[..., None], t * s.scale[:, None], 0)
    b = s.b.float().permute(0, 2, 1).reshape(count * rank, c["n"])
    out = torch.where(live[:, None], s.base + torch.matmul(t.reshape(n, count * rank), b), 0)
    return _round_rows(c["out"], out)


# ---- one pass: the library's operators -----------------------------------------


def _package():
    """This repository's package (its directory name contains a dot)."""
    if "nanochat_amd" not in sys.modules:
        pkg = os.path.join(_ROOT, "nanochatllms.cpp_amd")
        spec = importlib.util.spec_from_file_location("nanochat_amd", os.path.join(pkg, "__init__.py"),
                                                      submodule_search_locations=[pkg])
        mod = importlib.util.module_from_spec(spec)
        sys.modules["nanochat_amd"] = mod
        spec.loader.exec_module(mod)
    return sys.modules["nanochat_amd"]


class _Handles:
    """The descriptors and the workspace that a user's program keeps."""

    def __init__(self, s):
        nc, c = _package(), s.case
        nc.init(0)
        self.lib, self.check = nc.lib(), nc.check
        dtypes = {"q8": nc.Q8, "f16": nc.F16, "f32": nc.F32}
        ptr = lambda t: C.c_void_p(t.data_ptr() if t is not None else None)  # noqa: E731
        act = lambda kind, t, cols: nc.Tensor(t.data_ptr(), None, dtypes[kind], t.shape[0], cols,  # noqa: E731
                                              t.stride(0) * t.element_size())
        self.keep = []

        def ref(x):
            self.keep.append(x)
            return C.byref(x)

        if c["op"] == "lora":
            lora = nc.Lora(a=ptr(s.a), b=ptr(s.b), scale=ptr(s.scale), n_adapters=c["adapters"], rank=c["rank"],
                           k=c["k"], n=c["n"])
            self.args = (ref(act(c["rows"], s.x, c["k"])), ref(act("f32", s.base, c["n"])), ref(lora), ptr(s.adapter),
                         ptr(s.row_start), c["n_req"], s.max_new, ref(act(c["out"], s.out, c["n"])), None)
            return
        batch = ref(nc.PagedBatch(n_req=c["n_req"], max_tokens=s.max_tokens, max_pages=s.max_pages, max_new=s.max_new,
                                  max_kv=s.max_kv, new_len=ptr(s.new_len), seq_len=ptr(s.seq_len),
                                  block_table=ptr(s.table), row_start=ptr(s.row_start), kv_len=ptr(s.kv_len),
                                  positions=ptr(s.positions), slots=ptr(s.slots)))
        if c["op"] == "plan":
            pool = ref(nc.PagePool(free_pages=ptr(s.free_pages), state=ptr(s.pool), n_pages=s.n_pages,
                                   page_size=c["page"]))
            self.args = (pool, batch, None)
            return
        hq, d = c["hq"], c["d"]
        cache = ref(nc.PagedCache(k=ptr(s.kc), v=ptr(s.vc), k_deltas=ptr(s.kd), v_deltas=ptr(s.vd),
                                  dtype=dtypes[s.cache], n_pages=s.n_pages, page_size=c["page"], n_kv_heads=c["hkv"],
                                  d_head=d))
        if c["op"] == "append":
            q, k, v = (ref(act(c["rows"], x, h * d)) for x, h in ((s.q, hq), (s.k, c["hkv"]), (s.v, c["hkv"])))
            self.args = (q, k, v, ref(act(c["out"], s.q_out, hq * d)), cache, batch, ptr(s.rope), s.rope.shape[0],
                         s.rope.shape[1], None)
            return
        size = C.c_size_t()
        self.check(self.lib.nc_paged_attn_workspace(cache, batch, hq, c["window"], c["sink"], C.byref(size)),
                   "paged_attn_workspace")
        self.work = torch.empty(max(size.value, 16), dtype=torch.uint8, device="cuda")
        self.args = (ref(act(c["rows"], s.q, hq * d)), cache, batch, ref(act(c["rows"], s.out, hq * d)), hq,
                     c["window"], c["sink"], ptr(self.work), size.value, None)


def _run_own(s):
    if not hasattr(s, "handles"):
        s.handles = _Handles(s)
    h, c = s.handles, s.case
    if c["op"] == "plan":
        h.check(h.lib.nc_paged_plan(*h.args), "paged_plan")
        return s.row_start, s.kv_len, s.positions, s.slots, s.table, s.pool
    if c["op"] == "lora":
        h.check(h.lib.nc_lora_add(*h.args), "lora_add")
        if c["out"] != "q8":
            return s.out
        cols = _up(c["n"], 32) * 32
        return _read_rows("q8", s.out, cols)[:, :c["n"]].half()
    if c["op"] == "attn":
        h.check(h.lib.nc_paged_attn(*h.args), "paged_attn")
        return s.out if c["rows"] == "f16" else _read_rows("q8", s.out, c["hq"] * c["d"]).half()
    h.check(h.lib.nc_paged_append(*h.args), "paged_append")
    if c["out"] == "f16":
        return s.q_out, s.kc, s.vc
    live = s.slots[:s.tokens].long()
    at = (live // c["page"], slice(None), live % c["page"])
    return (_read_rows("q8", s.q_out, c["hq"] * c["d"]).half(), _values(s.kc[at], s.kd[at]).half(),
            _values(s.vc[at], s.vd[at]).half())


def run(state):
    if own:
        return _run_own(state)
    return {"plan": _plan, "append": _append, "attn": _attn, "lora": _lora}[state.case["op"]](state)


# ---- what a pass cannot do without -----------------------------------------------

_SIZE = {"q8": 34 / 32, "f16": 2.0, "f32": 4.0}


def work(case):
    c = case
    new, past = _lengths(c)
    tokens = sum(new)
    if c["op"] == "plan":
        fresh = sum(_up(n + p, c["page"]) - _up(p, c["page"]) for n, p in zip(new, past))
        return {"bytes": 4.0 * (4 * len(new) + 1 + 2 * tokens + 2 * fresh), "flops": 4.0 * tokens}
    if c["op"] == "lora":
        used = min(c["adapters"], len(new))
        return {"bytes": tokens * (c["k"] * _SIZE[c["rows"]] + c["n"] * (4 + _SIZE[c["out"]]))
                + 2.0 * used * c["rank"] * (c["k"] + c["n"]),
                "flops": 2.0 * tokens * c["rank"] * (c["k"] + c["n"])}
    d, hq, hkv = c["d"], c["hq"], c["hkv"]
    if c["op"] == "append":
        return {"bytes": tokens * d * (hq + 2 * hkv) * (_SIZE[c["rows"]] + _SIZE[c["out"]]),
                "flops": 3.0 * tokens * d * (hq + hkv)}
    pairs = keys = 0.0
    for n, p in zip(new, past):
        if not n:
            continue
        if not c["window"]:
            pairs += n * p + n * (n + 1) / 2
            keys += n + p
        else:
            w, k = c["window"], c["sink"]
            reach = [min(w, q + 1) + min(k, max(0, q + 1 - w)) for q in range(p, p + n)]
            pairs += sum(reach)
            lo = max(0, p + 1 - w)
            keys += n + p - lo + min(k, lo)
    return {"bytes": keys * hkv * d * 2 * _SIZE[c["cache"]] + 2 * tokens * hq * d * _SIZE[c["rows"]],
            "flops": 4.0 * pairs * hq * d}


# ---- the same in 64 bits -----------------------------------------------------------


def _exact_rows(kind, buf, cols):
    if kind != "q8":
        return buf.double()
    nb = cols // 32
    delta = buf[:, cols:cols + 2 * nb].contiguous().view(torch.float16).double()
    return buf[:, :cols].contiguous().view(torch.int8).double() * delta.repeat_interleave(32, 1)


def _exact_cache(codes, deltas, pages, count):
    """[position, kv head, d] of one request."""
    x = codes[pages].double()
    if deltas is not None:
        x = x * deltas[pages].double().repeat_interleave(32, -1)
    return x.transpose(1, 2).reshape(-1, x.shape[1], x.shape[3])[:count]


def _exact_q8(x):
    """The values of x's Q8 blocks: steps of a 127th of each block's largest magnitude."""
    blocks = x.reshape(-1, 32)
    step = blocks.abs().amax(1, keepdim=True) / 127
    count = (blocks.abs() / step.clamp(min=1e-300) + 0.5).floor() * blocks.sign()
    return (count * step.half().double()).reshape(x.shape)


def exact(case, seed):
    """The results from their definition; what Q8 rows hold of them where a result is stored as Q8."""
    c = case
    if c["op"] == "plan":
        return None
    s = prepare(case, seed)
    new, past = _lengths(c)
    n = s.max_tokens
    if c["op"] == "lora":
        x = _exact_rows(c["rows"], s.x, c["k"])
        out = torch.zeros(n, c["n"], dtype=torch.float64, device="cuda")
        at = 0
        for a, m in zip(s.adapter.tolist(), new):
            out[at:at + m] = s.base[at:at + m].double()
            if a >= 0 and m:
                low = x[at:at + m] @ s.a[a].double().T
                out[at:at + m] += s.scale[a].double() * (low @ s.b[a].double().T)
            at += m
        if c["out"] == "q8":
            out = _exact_q8(torch.nn.functional.pad(out, (0, -c["n"] % 32)))[:, :c["n"]]
        return out
    d, hq, hkv = c["d"], c["hq"], c["hkv"]
    if c["op"] == "append":
        q, k, v = (_exact_rows(c["rows"], x, h * d).reshape(n, h, d)[:s.tokens]
                   for x, h in ((s.q, hq), (s.k, hkv), (s.v, hkv)))
        pos = torch.cat([torch.arange(p, p + m, device="cuda") for m, p in zip(new, past)])
        half = s.rope.shape[1]
        turn = torch.complex(s.rope[..., 0].double(), s.rope[..., 1].double())[pos][:, None]

        def rotate(x):
            z = torch.complex(x[..., :half].contiguous(), x[..., half:2 * half].contiguous()) * turn
            return torch.cat([z.real, z.imag, x[..., 2 * half:]], -1)

        q = torch.nn.functional.pad(rotate(q).reshape(s.tokens, hq * d), (0, 0, 0, n - s.tokens))
        if c["out"] == "q8":
            return tuple(_exact_q8(x) for x in (q, rotate(k), v))
        caches = [torch.zeros(s.kc.shape, dtype=torch.float64, device="cuda") for _ in range(2)]
        slot = s.slots[:s.tokens].long()
        for cache, x in zip(caches, (rotate(k), v)):
            cache[slot // c["page"], :, slot % c["page"]] = x
        return (q, *caches)
    q = _exact_rows(c["rows"], s.q, hq * d).reshape(n, hq, d)
    out = torch.zeros(n, hq, d, dtype=torch.float64, device="cuda")
    at = 0
    for r, (m, p) in enumerate(zip(new, past)):
        if not m:
            continue
        pages = s.table[r, :_up(m + p, c["page"])].long()
        k, v = (_exact_cache(x, y, pages, m + p) for x, y in ((s.kc, s.kd), (s.vc, s.vd)))
        key, row = torch.arange(m + p, device="cuda")[None], torch.arange(p, p + m, device="cuda")[:, None]
        hidden = key > row
        if c["window"]:
            hidden |= (row - key >= c["window"]) & (key >= c["sink"])
        for h in range(hq):
            j = h // (hq // hkv)
            sc = (q[at:at + m, h] @ k[:, j].T.contiguous()) / d ** 0.5
            out[at:at + m, h] = torch.softmax(sc.masked_fill(hidden, -math.inf), -1) @ v[:, j].contiguous()
        at += m
    out = out.reshape(n, hq * d)
    return _exact_q8(out) if c["rows"] == "q8" else out
