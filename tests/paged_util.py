"""Requests, pages and plain 64-bit forms for the tests of batched serving."""
import ctypes as C
import math

import torch

from nc_pkg import nc

DT = {"f16": nc.F16, "q8": nc.Q8, "f32": nc.F32}
HALF = 2.0 ** -11  # half a step of fp16, relative
TINY = 2.0 ** -25  # half of fp16's smallest step


def up(a, b):
    return -(-a // b)


def ptr(t):
    return C.c_void_p(t.data_ptr() if t is not None else None)


def ints(v, device="cuda"):
    return torch.tensor(v, dtype=torch.int32, device=device)


def stream(s):
    return C.c_void_p(s.cuda_stream)


def sync():
    torch.cuda.synchronize()


def q8_parts(x):
    """Codes (as doubles) and fp16 deltas of blocks of 32 along the last axis, as q8_quantize makes them."""
    b = x.float().reshape(*x.shape[:-1], -1, 32)
    delta = b.abs().amax(-1, keepdim=True) / 127
    q = b * torch.where(delta > 0, 1 / delta, torch.zeros_like(delta))
    q = torch.sign(q) * torch.floor(q.abs().double() + 0.5)
    return q.reshape(x.shape), delta[..., 0].half()


def q8_values(q, delta):
    return (q.double().reshape(*q.shape[:-1], -1, 32) * delta.double()[..., None]).reshape(q.shape)


class Rows:
    """Activation rows on the GPU in the library's layout, filled with `fill` bytes where no value goes."""

    def __init__(self, kind, n, cols, values=None, fill=0, extra_pitch=0):
        self.kind, self.n, self.cols = kind, n, cols
        self.pitch = nc.lib().nc_act_pitch(DT[kind], cols) + extra_pitch
        self.buf = torch.full((max(n, 1), self.pitch), fill, dtype=torch.uint8, device="cuda")
        self.t = nc.Tensor(self.buf.data_ptr(), None, DT[kind], n, cols, self.pitch)
        self.ref = C.byref(self.t)
        if values is not None and n:
            values = values.cuda()
            if kind == "q8":
                nb = up(cols, 32)
                q, d = q8_parts(torch.nn.functional.pad(values, (0, nb * 32 - cols)))
                self.buf[:n, :nb * 32] = q.to(torch.int8).view(torch.uint8)
                self.buf[:n, nb * 32:nb * 34] = d.contiguous().view(torch.uint8)
            else:
                v = values.half() if kind == "f16" else values.float()
                self.buf[:n, :cols * v.element_size()] = v.contiguous().view(torch.uint8)

    def values(self):
        """What the rows stand for, in 64 bits on the host."""
        b = self.buf[:self.n].cpu()
        if self.kind == "q8":
            nb = up(self.cols, 32)
            return q8_values(b[:, :nb * 32].contiguous().view(torch.int8),
                             b[:, nb * 32:nb * 34].contiguous().view(torch.float16))[:, :self.cols]
        t, size = (torch.float16, 2) if self.kind == "f16" else (torch.float32, 4)
        return b[:, :self.cols * size].contiguous().view(t).double()


class Cache:
    def __init__(self, kind, n_pages, page, hkv, d, fill=0):
        self.kind, self.shape = kind, (n_pages, hkv, page, d)
        if kind == "f16":
            self.k, self.v = (torch.full(self.shape, fill, dtype=torch.float16, device="cuda") for _ in range(2))
            self.kd = self.vd = None
        else:
            self.k, self.v = (torch.zeros(self.shape, dtype=torch.int8, device="cuda") for _ in range(2))
            self.kd, self.vd = (torch.full((n_pages, hkv, page, d // 32), fill, dtype=torch.float16, device="cuda")
                                for _ in range(2))
        self.t = nc.PagedCache(k=ptr(self.k), v=ptr(self.v), k_deltas=ptr(self.kd), v_deltas=ptr(self.vd),
                               dtype=DT[kind], n_pages=n_pages, page_size=page, n_kv_heads=hkv, d_head=d)
        self.ref = C.byref(self.t)

    def put(self, which, slots, x):
        """x [n, hkv, d] into the slots."""
        n_pages, hkv, page, d = self.shape
        x, slots = x.cuda(), torch.as_tensor(slots, device="cuda").long()
        at = (slots // page, slice(None), slots % page)
        if self.kind == "f16":
            getattr(self, which)[at] = x.half()
        else:
            q, delta = q8_parts(x)
            getattr(self, which)[at] = q.to(torch.int8)
            getattr(self, which + "d")[at] = delta

    def values(self, which, slots):
        n_pages, hkv, page, d = self.shape
        slots = torch.as_tensor(slots, device="cuda").long()
        at = (slots // page, slice(None), slots % page)
        x = getattr(self, which)[at].cpu()
        return x.double() if self.kind == "f16" else q8_values(x, getattr(self, which + "d")[at].cpu())


class Step:
    """One step's requests over a pool in random order, with the tables that nc_paged_plan makes."""

    def __init__(self, new, past, page, g, pad=0, spare=5, max_new=None, max_kv=None, first_page=0, fill=-7):
        self.new, self.past, self.page, self.n_req = list(new), list(past), page, len(new)
        self.tokens = sum(new)
        self.max_tokens = self.tokens + pad
        self.max_new = max(new) if max_new is None else max_new
        self.max_kv = max(n + p for n, p in zip(new, past)) if max_kv is None else max_kv
        self.max_pages = max(1, up(self.max_kv, page)) + 1
        have = [up(p, page) for p in past]
        need = [up(p + n, page) for n, p in zip(new, past)]
        self.n_pages = first_page + sum(need) + spare
        order = (torch.randperm(self.n_pages - first_page, generator=g) + first_page).tolist()
        self.table_before = [[-1] * self.max_pages for _ in new]
        for r, h in enumerate(have):
            for j in range(h):
                self.table_before[r][j] = order.pop()
        self.free_before = list(order)
        self.plan_on_host(have, need)
        dev = lambda v, n: ints(v if v is not None else [fill] * n)  # noqa: E731
        self.new_len, self.seq_len = ints(self.new), ints(self.past)
        self.table = ints(self.table_before)
        self.free_pages = ints(self.free_before + [fill] * (self.n_pages - len(self.free_before)))
        self.state = ints([len(self.free_before), fill, fill, 0])
        self.row_start, self.kv_len = dev(None, self.n_req + 1), dev(None, self.n_req)
        self.positions, self.slots = dev(None, max(1, self.max_tokens)), dev(None, max(1, self.max_tokens))
        self.describe()

    def plan_on_host(self, have, need):
        free = list(self.free_before)
        self.want_table = [list(t) for t in self.table_before]
        self.want_pos, self.want_slots, self.want_rows = [], [], [0]
        for r, (n, p) in enumerate(zip(self.new, self.past)):
            for j in range(have[r], need[r]):
                self.want_table[r][j] = free.pop()
            for i in range(p, p + n):
                self.want_pos.append(i)
                self.want_slots.append(self.want_table[r][i // self.page] * self.page + i % self.page)
            self.want_rows.append(self.want_rows[-1] + n)
        pad = [-1] * (self.max_tokens - self.tokens)
        self.want_pos += pad
        self.want_slots += pad
        self.want_free = free

    def describe(self):
        self.pool = nc.PagePool(free_pages=ptr(self.free_pages), state=ptr(self.state), n_pages=self.n_pages,
                                page_size=self.page)
        self.batch = nc.PagedBatch(n_req=self.n_req, max_tokens=self.max_tokens, max_pages=self.max_pages,
                                   max_new=self.max_new, max_kv=self.max_kv, new_len=ptr(self.new_len),
                                   seq_len=ptr(self.seq_len), block_table=ptr(self.table),
                                   row_start=ptr(self.row_start), kv_len=ptr(self.kv_len),
                                   positions=ptr(self.positions), slots=ptr(self.slots))
        self.pool_ref, self.ref = C.byref(self.pool), C.byref(self.batch)

    def planned(self):
        """The tables as a plan leaves them, without running one."""
        self.table.copy_(ints(self.want_table))
        self.row_start.copy_(ints(self.want_rows))
        self.kv_len.copy_(ints([n + p for n, p in zip(self.new, self.past)]))
        if self.max_tokens:
            self.positions.copy_(ints(self.want_pos))
            self.slots.copy_(ints(self.want_slots))
        return self

    def past_slots(self, r):
        return [self.want_table[r][i // self.page] * self.page + i % self.page for i in range(self.past[r] + self.new[r])]


def workspace(step, cache, hq, window, sink):
    size = C.c_size_t()
    nc.check(nc.lib().nc_paged_attn_workspace(cache.ref, step.ref, hq, window, sink, C.byref(size)), "workspace")
    # NaN bytes: nothing may come from what lies there
    return torch.full((max(size.value, 16),), 0xFF, dtype=torch.uint8, device="cuda"), size.value


def attend(step, cache, q, out, hq, window=0, sink=0, work=None, on=None):
    work = work or workspace(step, cache, hq, window, sink)
    nc.check(nc.lib().nc_paged_attn(q.ref, cache.ref, step.ref, out.ref, hq, window, sink, ptr(work[0]), work[1], on),
             "paged_attn")


def visible(p, kv, window, sink):
    j = torch.arange(kv)
    seen = j <= p
    return seen & ((j > p - window) | (j < sink)) if window else seen


def plain_attention(step, cache, q, hq, window=0, sink=0, hidden=None):
    """64-bit results [tokens, hq * d] and, for each value, how far the kernel's documented roundings can take it.

    Over an fp16 cache, to first order: a probability's rounding to fp16 (HALF of itself) and, of Q8 q rows, that of the
    scores (HALF of sum |q k| / sqrt d), which changes a weight by its difference from the row's mean change.  Over a Q8
    cache nothing enters rounded.  fp32 sums and exp2 of a few hundred terms are held to 2^-16 of the terms' magnitudes,
    scores to 2^-20."""
    n_pages, hkv, page, d = cache.shape
    group = hq // hkv
    eps_p = HALF if cache.kind == "f16" else 0.0
    eps_q = HALF if cache.kind == "f16" and q.kind == "q8" else 0.0
    qv = q.values().reshape(-1, hq, d)
    out = torch.zeros(step.tokens, hq, d, dtype=torch.float64)
    tol = torch.zeros_like(out)
    for r in range(step.n_req):
        n, p, first = step.new[r], step.past[r], step.want_rows[r]
        if not n:
            continue
        slots = step.past_slots(r)
        k, v = cache.values("k", slots), cache.values("v", slots)
        for i in range(n):
            seen = visible(p + i, p + n, window, sink)
            if hidden is not None:
                seen &= ~hidden[r]
            if not seen.any():
                continue
            kk, vv = k[seen].repeat_interleave(group, 1), v[seen].repeat_interleave(group, 1)
            s = torch.einsum("hd,jhd->hj", qv[first + i], kk) / math.sqrt(d)
            mag = torch.einsum("hd,jhd->hj", qv[first + i].abs(), kk.abs()) / math.sqrt(d)
            w = torch.softmax(s, -1)
            out[first + i] = torch.einsum("hj,jhd->hd", w, vv)
            weight = torch.einsum("hj,jhd->hd", w, vv.abs())
            ds = (mag * (eps_q + 2.0 ** -20)).amax(-1, keepdim=True)
            tol[first + i] = weight * (eps_p + 2 * ds + 2.0 ** -16) + TINY
    return out.reshape(step.tokens, hq * d), tol.reshape(step.tokens, hq * d)


def rounded(kind, x, tol):
    """The tolerance of a result once stored: fp16 rounds by half a step; a Q8 code too, of its block's step, which
    follows the block's largest value, and the step itself rounds to fp16."""
    if kind == "f32":
        return tol + x.abs() * 2.0 ** -23
    if kind == "f16":
        return tol + (x.abs() + tol) * HALF + TINY
    pad = -x.shape[-1] % 32
    blocks = lambda t: torch.nn.functional.pad(t, (0, pad)).reshape(*t.shape[:-1], -1, 32)  # noqa: E731
    top = (blocks(x).abs() + blocks(tol)).amax(-1, keepdim=True)
    # the code rounds by half a step; the kept step is off by HALF of itself (TINY where it is subnormal), 127 of them
    # at most; a quarter of a step's 2^-10 for the fp32 product that is rounded
    step = top / 127 * (0.5 + 2.0 ** -12) + 127 * (top / 127 * HALF + TINY)
    return tol + step.expand(*step.shape[:-1], 32).reshape(*x.shape[:-1], -1)[..., :x.shape[-1]]


def within(got, want, tol, what=""):
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} values off, worst "
                           f"{((got - want).abs() / tol)[bad].max():.3g} times the tolerance, first at "
                           f"{bad.nonzero()[0].tolist()}: {got[bad][0]} for {want[bad][0]}")
