"""nc_lora_add against the formula in 64 bits."""
import ctypes as C

import pytest
import torch

import paged_util as P
from paged_util import Rows, ints, rounded, sync, within

pytestmark = pytest.mark.gpu


def make(gpu, n_adapters, rank, k, n, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    a = (torch.randn(n_adapters, rank, k, generator=g) * k ** -0.5).half().cuda()
    b = (torch.randn(n_adapters, n, rank, generator=g) * scale).half().cuda()
    s = torch.rand(n_adapters, generator=g).cuda() + 0.5
    t = gpu.Lora(a=P.ptr(a), b=P.ptr(b), scale=P.ptr(s), n_adapters=n_adapters, rank=rank, k=k, n=n)
    return (a, b, s, t), g


def want_of(lora, x, base, starts, adapters, max_new):
    """64-bit results and the error that fp32 sums can make of them.

    t = x a^T sums k fp32 products (k/32 matrix steps, the codes' sums exact: k 2^-24 of the magnitudes bounds any
    order), is then held to 2^-22 of the row's largest, and the second sum of 2 * rank products and the base add
    another (2 rank + 2) 2^-24 of its magnitudes."""
    a, b, s, t = lora
    x, base = x.values(), base.values()
    out, tol = base.clone(), torch.zeros_like(base)
    for r, ad in enumerate(adapters):
        rows = slice(starts[r], min(starts[r + 1], starts[r] + max_new))
        if not 0 <= ad < a.shape[0]:
            continue
        ad_a, ad_b, sc = a[ad].cpu().double(), b[ad].cpu().double(), s[ad].item()
        low, mag = x[rows] @ ad_a.T, x[rows].abs() @ ad_a.abs().T
        out[rows] += sc * (low @ ad_b.T)
        err = mag * t.k * 2.0 ** -24 + (low.abs().amax(1, keepdim=True) if low.numel() else low) * 2.0 ** -22
        tol[rows] = sc * (err @ ad_b.abs().T) + (2 * t.rank + 2) * 2.0 ** -24 * (
            sc * (low.abs() @ ad_b.abs().T) + base[rows].abs())
    return out, tol


def add(gpu, x, base, lora, adapters, starts, max_new, out, on=None):
    a, s = ints(adapters), ints(starts)
    gpu.check(gpu.lib().nc_lora_add(x.ref, base.ref, C.byref(lora[3]), P.ptr(a), P.ptr(s), len(adapters), max_new, out.ref,
                                    on), "lora_add")
    return a, s


CASES = [
    # (rows, out, rank, k, n, new rows, adapters)
    ("f16", "f32", 16, 64, 128, [1], [0]),
    ("f16", "f16", 16, 2048, 2560, [1] * 5, [2, -1, 0, 2, 1]),
    ("q8", "f32", 16, 2048, 96, [1, 0, 3], [0, 1, 2]),
    ("q8", "q8", 8, 1280, 1000, [4, 17], [1, 0]),
    ("f16", "q8", 32, 96, 33, [16, 1, 15], [0, 0, 0]),
    ("f16", "f32", 1, 32, 1, [2, 2], [0, 2]),
    ("q8", "f32", 5, 160, 7, [31, 33], [2, 2]),
    ("f16", "f16", 24, 224, 130, [100], [1]),
    ("q8", "f16", 64, 2304, 515, [40, 1, 70], [0, 1, 3]),
    ("f16", "f32", 100, 320, 260, [33], [1]),
    ("q8", "q8", 128, 512, 2048, [50, 9], [2, 0]),
    ("f16", "f32", 128, 5632, 64, [20], [2]),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c[:5])))
def test_lora(gpu, case):
    rows, okind, rank, k, n, new, adapters = case
    lora, g = make(gpu, 3, rank, k, n, seed=rank + n)
    starts = [sum(new[:r]) for r in range(len(new) + 1)]
    total = starts[-1] + 3  # rows behind the last request
    x = Rows(rows, total, k, torch.randn(total, k, generator=g))
    base = Rows("f32", total, n, torch.randn(total, n, generator=g))
    out = Rows(okind, total, n, fill=0x3C)
    add(gpu, x, base, lora, adapters, starts, max(new), out)
    sync()
    want, tol = want_of(lora, x, base, starts, adapters, max(new))
    live = slice(0, starts[-1])
    within(out.values()[live], want[live], rounded(okind, want[live], tol[live]), str(case))
    assert (out.buf[starts[-1]:] == 0x3C).all()
    for r, ad in enumerate(adapters):  # a request of the model itself: the base as it is
        if not 0 <= ad < 3 and okind == "f32":
            assert torch.equal(out.buf[starts[r]:starts[r + 1]], base.buf[starts[r]:starts[r + 1]])


@pytest.mark.parametrize("rows", ["f16", "q8"])
def test_in_place_many_requests_and_again(gpu, rows):
    new = [(7 * i) % 5 for i in range(300)]
    starts = [sum(new[:r]) for r in range(len(new) + 1)]
    adapters = [(i * 5) % 9 - 1 for i in range(300)]
    lora, g = make(gpu, 8, 16, 128, 200, seed=3)
    total = starts[-1]
    x = Rows(rows, total, 128, torch.randn(total, 128, generator=g))
    values = torch.randn(total, 200, generator=g)
    base, out = Rows("f32", total, 200, values), Rows("f32", total, 200)
    add(gpu, x, base, lora, adapters, starts, 4, out)
    sync()
    want, tol = want_of(lora, x, base, starts, adapters, 4)
    within(out.values(), want, rounded("f32", want, tol))
    add(gpu, x, base, lora, adapters, starts, 4, base)
    sync()
    assert torch.equal(base.buf, out.buf)


def test_range_of_the_low_rank_products(gpu):
    """Products far beyond fp16's largest and far below its smallest are as exact as others."""
    for size in (2.0 ** 12, 1.0, 2.0 ** -9):
        lora, g = make(gpu, 1, 16, 2048, 64, seed=4, scale=size)
        x = Rows("f16", 4, 2048, torch.randn(4, 2048, generator=g) * size * 4)
        a = lora[0]
        a.mul_(size * 4)
        base = Rows("f32", 4, 64, torch.zeros(4, 64))
        out = Rows("f32", 4, 64)
        add(gpu, x, base, lora, [0], [0, 4], 4, out)
        sync()
        want, tol = want_of(lora, x, base, [0, 4], [0], 4)
        within(out.values(), want, rounded("f32", want, tol), f"size {size}")


def test_rows_that_are_zero_or_not_finite(gpu):
    lora, g = make(gpu, 1, 16, 64, 96, seed=5)
    v = torch.randn(4, 64, generator=g)
    v[0], v[2, 7], v[3, 9] = 0.0, float("nan"), float("inf")
    x, base = Rows("f16", 4, 64, v), Rows("f32", 4, 96, torch.randn(4, 96, generator=g))
    out = Rows("f32", 4, 96)
    add(gpu, x, base, lora, [0], [0, 4], 4, out)
    sync()
    got = out.values()
    assert torch.equal(got[0], base.values()[0])
    want, tol = want_of(lora, x, base, [0, 4], [0], 4)
    within(got[1], want[1], rounded("f32", want[1], tol[1]))
    assert got[2].isnan().all() and not got[3].isfinite().any()


def test_max_new_bounds_each_request(gpu):
    lora, g = make(gpu, 2, 8, 32, 40, seed=6)
    starts = [0, 20, 23, 60]
    x, base = Rows("f16", 60, 32, torch.randn(60, 32, generator=g)), Rows("f32", 60, 40, torch.randn(60, 40, generator=g))
    out = Rows("f32", 60, 40, fill=0x3C)
    add(gpu, x, base, lora, [0, -1, 1], starts, 18, out)
    sync()
    want, tol = want_of(lora, x, base, starts, [0, -1, 1], 18)
    done = torch.zeros(60, dtype=torch.bool)
    for r in range(3):
        done[starts[r]:min(starts[r + 1], starts[r] + 18)] = True
    within(out.values()[done], want[done], rounded("f32", want[done], tol[done]))
    assert (out.buf[~done.cuda()] == 0x3C).all()


def test_row_starts_that_lead_nowhere(gpu):
    lora, g = make(gpu, 1, 16, 64, 32, seed=7)
    x = Rows("f16", 6, 64, torch.randn(6, 64, generator=g))
    base = Rows("f32", 6, 32, torch.randn(6, 32, generator=g))
    big = 2 ** 31 - 1
    for starts in ([0, -5, 4, 6], [big] * 4, [-big, big, 0, 3], [6, 5, 2, 0]):
        whole = torch.full((14, 128), 0x3C, dtype=torch.uint8, device="cuda")
        t = gpu.Tensor(whole[4:].data_ptr(), None, gpu.F32, 6, 32, 128)
        keep = ints([0, 0, 0]), ints(starts)
        gpu.check(gpu.lib().nc_lora_add(x.ref, base.ref, C.byref(lora[3]), P.ptr(keep[0]), P.ptr(keep[1]), 3, 6,
                                        C.byref(t), None), "lora_add")
        sync()
        assert (whole[:4] == 0x3C).all() and (whole[10:] == 0x3C).all()


def test_captured_and_on_another_stream(gpu):
    lora, g = make(gpu, 4, 16, 256, 300, seed=8)
    x = Rows("q8", 40, 256, torch.randn(40, 256, generator=g))
    base, out = Rows("f32", 40, 300, torch.randn(40, 300, generator=g)), Rows("f32", 40, 300)
    adapter, starts = ints([0, 1, 2, 3]), ints([0, 10, 20, 30, 40])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        gpu.check(gpu.lib().nc_lora_add(x.ref, base.ref, C.byref(lora[3]), P.ptr(adapter), P.ptr(starts), 4, 40, out.ref,
                                        P.stream(torch.cuda.current_stream())), "lora_add")
    for ad, st in (([0, 1, 2, 3], [0, 10, 20, 30, 40]), ([3, -1, 0, 0], [0, 1, 1, 5, 40]), ([1, 1, 1, 9], [0, 40, 40, 40, 40])):
        adapter.copy_(ints(ad))
        starts.copy_(ints(st))
        graph.replay()
        sync()
        want, tol = want_of(lora, x, base, st, ad, 40)
        within(out.values(), want, rounded("f32", want, tol))
