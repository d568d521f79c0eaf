"""The operators of batched serving together, over several steps of several requests.

Each step plans, projects the step's rows with nc_matmul_2d, adds adapters, appends, attends and commits; between steps
one request ends, its pages go to another, and a prompt comes in chunks.  At every step each request's cached rows must
be, bit for bit, what nc_matmul_2d and nc_rotary_emb give for the whole sequence at once, and the attention's rows what
the formula gives over them."""
import ctypes as C

import numpy as np
import pytest
import torch

import paged_util as P
from paged_util import Cache, Rows, ints, plain_attention, rounded, sync, within, workspace

pytestmark = pytest.mark.gpu

DM, HQ, HKV, D, PAGE, PAGES = 256, 4, 2, 64, 16, 24


class Weight:
    def __init__(self, gpu, kind, rows, cols, g):
        L, dt = gpu.lib(), {"f16": gpu.F16, "q8": gpu.Q8}[kind]
        cb, db = C.c_size_t(), C.c_size_t()
        gpu.check(L.nc_weight_bytes(dt, rows, cols, C.byref(cb), C.byref(db)))
        self.codes = torch.zeros(cb.value, dtype=torch.uint8, device="cuda")
        self.deltas = torch.zeros(max(db.value, 16), dtype=torch.uint8, device="cuda")
        w = (torch.randn(rows, cols, generator=g) * 0.1).cuda()
        self.t = gpu.Tensor(self.codes.data_ptr(), self.deltas.data_ptr() if db.value else None, dt, rows, cols, 0)
        self.ref = C.byref(self.t)
        sync()
        gpu.check(L.nc_weight_quantize(P.ptr(w), self.ref, None))
        gpu.check(L.nc_synchronize())


def matmul(gpu, x, w, n):
    out = Rows("f32", n, w.t.rows)
    gpu.check(gpu.lib().nc_matmul_2d(x.ref, w.ref, out.ref, 0, n, None), "matmul_2d")
    return out


class Server:
    """What a program keeps between steps; `seen` stands in for it in plain_attention."""

    def __init__(self, gpu, kind, n_req, max_tokens):
        self.n_req, self.max_tokens, self.max_pages, self.max_new, self.max_kv = n_req, max_tokens, 9, 40, 140
        self.free, self.state = ints([0] * PAGES), ints([0] * 4)
        self.new_len, self.seq_len, self.kv_len = (ints([0] * n_req) for _ in range(3))
        self.table, self.row_start = ints([[-1] * self.max_pages] * n_req), ints([0] * (n_req + 1))
        self.positions, self.slots = ints([-1] * max_tokens), ints([-1] * max_tokens)
        self.finished = ints([0] * n_req)
        self.pool = gpu.PagePool(free_pages=P.ptr(self.free), state=P.ptr(self.state), n_pages=PAGES, page_size=PAGE)
        self.batch = gpu.PagedBatch(n_req=n_req, max_tokens=max_tokens, max_pages=self.max_pages, max_new=self.max_new,
                                    max_kv=self.max_kv, new_len=P.ptr(self.new_len), seq_len=P.ptr(self.seq_len),
                                    block_table=P.ptr(self.table), row_start=P.ptr(self.row_start),
                                    kv_len=P.ptr(self.kv_len), positions=P.ptr(self.positions), slots=P.ptr(self.slots))
        self.ref, self.pool_ref = C.byref(self.batch), C.byref(self.pool)
        gpu.check(gpu.lib().nc_page_pool_init(self.pool_ref, None))

    def facts(self, new, past):
        """The step as paged_util's plain forms take it, read back from the tables."""
        self.new, self.past, self.tokens = new, past, sum(new)
        self.want_rows = self.row_start.tolist()
        table = self.table.tolist()
        self.past_slots = lambda r: [table[r][i // PAGE] * PAGE + i % PAGE for i in range(past[r] + new[r])]


@pytest.mark.parametrize("kind", ["f16", "q8"])
@pytest.mark.parametrize("window,sink", [(0, 0), (20, 2)])
def test_steps(gpu, kind, window, sink):
    L = gpu.lib()
    g = torch.Generator().manual_seed(21)
    wq, wk, wv, wo = (Weight(gpu, kind, r, c, g) for r, c in
                      ((HQ * D, DM), (HKV * D, DM), (HKV * D, DM), (DM, HQ * D)))
    a = (torch.randn(3, 8, DM, generator=g) * 0.1).half().cuda()
    b = (torch.randn(3, HQ * D, 8, generator=g) * 0.1).half().cuda()
    scale = torch.tensor([1.0, 0.5, 2.0], device="cuda")
    lora = gpu.Lora(a=P.ptr(a), b=P.ptr(b), scale=P.ptr(scale), n_adapters=3, rank=8, k=DM, n=HQ * D)
    adapters = [2, -1, 0, 2]
    adapter = ints(adapters)
    rope = np.zeros((140, D // 2, 2), np.float32)
    gpu.check(L.nc_rope_table(140, D, 1.0, rope.ctypes.data_as(C.c_void_p)))
    rope = torch.from_numpy(rope).cuda()
    sv = Server(gpu, kind, 4, 96)
    cache = Cache(kind, PAGES, PAGE, HKV, D, fill=float("nan"))
    work = workspace(sv, cache, HQ, window, sink)
    history = [torch.zeros(0, DM) for _ in range(4)]
    steps = [([37, 5, 0, 1], []), ([40, 1, 3, 1], []), ([1, 1, 1, 1], [0]), ([33, 1, 40, 1], [1, 3]), ([1, 40, 1, 0], []),
             ([1, 1, 1, 19], [])]
    done = []
    for step, (new, finished) in enumerate(steps):
        past = [len(h) for h in history]
        x = torch.randn(96, DM, generator=g)
        sv.new_len.copy_(ints(new))
        sv.finished.copy_(ints([int(r in finished) for r in range(4)]))
        xr = Rows(kind, 96, DM, x)
        q, k, v = (matmul(gpu, xr, w, 96) for w in (wq, wk, wv))
        plain_q = Rows("f32", 96, HQ * D, q.values().float())
        sync()
        gpu.check(L.nc_paged_plan(sv.pool_ref, sv.ref, None), "plan")
        gpu.check(L.nc_lora_add(xr.ref, q.ref, C.byref(lora), P.ptr(adapter), P.ptr(sv.row_start), 4, sv.max_new, q.ref,
                                None), "lora")
        qr, att = Rows(kind, 96, HQ * D), Rows(kind, 96, HQ * D)
        gpu.check(L.nc_paged_append(q.ref, k.ref, v.ref, qr.ref, cache.ref, sv.ref, P.ptr(rope), 140, D // 2, None),
                  "append")
        gpu.check(L.nc_paged_attn(qr.ref, cache.ref, sv.ref, att.ref, HQ, window, sink, P.ptr(work[0]), work[1], None),
                  "attn")
        y = matmul(gpu, att, wo, 96)
        sync()
        assert sv.state[2].item() == 0
        sv.facts(new, past)
        # adapters: 64 bits from the rows that the projection read
        xv, want_q, tol_q = xr.values(), plain_q.values(), torch.zeros(96, HQ * D, dtype=torch.float64)
        for r, ad in enumerate(adapters):
            rows = slice(sv.want_rows[r], sv.want_rows[r + 1])
            if ad >= 0:
                low = xv[rows] @ a[ad].cpu().double().T
                bb, sc = b[ad].cpu().double(), scale[ad].item()
                want_q[rows] += sc * (low @ bb.T)
                err = (xv[rows].abs() @ a[ad].cpu().double().abs().T) * (DM * 2.0 ** -24) + 2.0 ** -22 * (
                    low.abs().amax(1, keepdim=True) if low.numel() else 0)
                tol_q[rows] = sc * (err @ bb.abs().T) + 18 * 2.0 ** -24 * (sc * (low.abs() @ bb.abs().T) + want_q[rows].abs())
        live = slice(0, sv.tokens)
        within(q.values()[live], want_q[live], rounded("f32", want_q[live], tol_q[live]), f"adapters, step {step}")
        # the cache: every position of every request, as one sequence gives them
        for r in range(4):
            history[r] = torch.cat([history[r], x[sv.want_rows[r]:sv.want_rows[r + 1]]])
            n = len(history[r])
            if not n:
                continue
            whole = Rows(kind, n, DM, history[r])
            kk, vv = matmul(gpu, whole, wk, n), matmul(gpu, whole, wv, n)
            turned = Rows("f32", n, HKV * D)
            gpu.check(L.nc_rotary_emb(kk.ref, turned.ref, D, 1.0, P.ptr(rope), 0, n, None), "rotary_emb")
            sync()
            for name, rows in (("k", turned), ("v", vv)):
                want = Rows(kind, n, HKV * D, rows.values().float()).values()
                assert torch.equal(cache.values(name, sv.past_slots(r)).reshape(n, -1), want), (step, r, name)
        want, tol = plain_attention(sv, cache, qr, HQ, window, sink)
        within(att.values()[live], want, rounded(kind, want, tol), f"attention, step {step}")
        assert torch.isfinite(y.values()[live]).all()
        gpu.check(L.nc_paged_commit(sv.pool_ref, sv.ref, P.ptr(sv.finished), None), "commit")
        sync()
        for r in finished:
            done.append(len(history[r]))
            history[r] = torch.zeros(0, DM)
        held = sum(P.up(len(h), PAGE) for h in history)
        assert sv.seq_len.tolist() == [len(h) for h in history] and sv.state[0].item() == PAGES - held
    assert done == [78, 8, 4]  # 37 + 40 + 1, 5 + 1 + 1 + 1 and 1 + 1 + 1 + 1 rows


@pytest.mark.parametrize("kind", ["f16", "q8"])
def test_a_captured_step_replayed_with_other_lengths(gpu, kind):
    """One graph for every step, under bounds that hold them all: single tokens, chunks on both kinds of tiles, a step
    that does not fit, requests that end."""
    L = gpu.lib()
    g = torch.Generator().manual_seed(22)
    sv = Server(gpu, kind, 4, 96)
    cache = Cache(kind, PAGES, PAGE, HKV, D, fill=float("nan"))
    work = workspace(sv, cache, HQ, 0, 0)
    q, k, v = (Rows("f32", 96, n) for n in (HQ * D, HKV * D, HKV * D))
    qr, att = Rows(kind, 96, HQ * D), Rows(kind, 96, HQ * D, fill=0x3C)
    graph = torch.cuda.CUDAGraph()
    sync()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        on = P.stream(torch.cuda.current_stream())
        gpu.check(L.nc_paged_plan(sv.pool_ref, sv.ref, on), "plan")
        gpu.check(L.nc_paged_append(q.ref, k.ref, v.ref, qr.ref, cache.ref, sv.ref, None, 0, 0, on), "append")
        gpu.check(L.nc_paged_attn(qr.ref, cache.ref, sv.ref, att.ref, HQ, 0, 0, P.ptr(work[0]), work[1], on), "attn")
        gpu.check(L.nc_paged_commit(sv.pool_ref, sv.ref, P.ptr(sv.finished), on), "commit")
    past, fitted = [0] * 4, []
    for new, finished in (([40, 1, 0, 9], []), ([1, 1, 1, 1], []), ([40, 40, 3, 1], []), ([0, 41, 0, 0], []),
                          ([20, 30, 40, 6], []), ([1, 1, 1, 1], [1]), ([1, 40, 1, 40], []), ([0, 0, 0, 0], [0, 3]),
                          ([30, 0, 30, 2], []), ([1, 1, 1, 1], [])):
        sv.new_len.copy_(ints(new))
        sv.finished.copy_(ints([int(r in finished) for r in range(4)]))
        for rows in (q, k, v):
            rows.buf.view(torch.float32).copy_(torch.randn(96, rows.cols, generator=g))
        before = att.buf.clone()
        sync()
        table = sv.table.tolist()  # requests that end here do so in steps that take no new page of theirs
        graph.replay()
        sync()
        status = sv.state[2].item()
        fitted.append(status == 0)
        if status:
            assert torch.equal(att.buf, before) and sv.seq_len.tolist() == past
            continue
        sv.facts(new, past)
        after = sv.table.tolist()
        assert all(after[r] == [-1] * sv.max_pages for r in finished)
        tables = [table[r] if r in finished else after[r] for r in range(4)]
        sv.past_slots = lambda r: [tables[r][i // PAGE] * PAGE + i % PAGE for i in range(past[r] + new[r])]
        if sv.tokens:
            want, tol = plain_attention(sv, cache, qr, HQ)
            within(att.values()[:sv.tokens], want, rounded(kind, want, tol), f"{new} after {past}")
        assert torch.equal(att.buf[sv.tokens:], before[sv.tokens:])
        past = [0 if r in finished else p + n for r, (p, n) in enumerate(zip(past, new))]
        assert sv.seq_len.tolist() == past
    assert fitted == [True, True, True, False, True, True, True, True, True, True]
