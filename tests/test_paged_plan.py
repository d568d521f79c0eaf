"""nc_paged_plan, nc_paged_commit and nc_page_pool_init against a page allocator in Python: every integer equal."""
import ctypes as C

import pytest
import torch

import paged_util as P
from paged_util import Step, ints, sync

pytestmark = pytest.mark.gpu


def plan(gpu, s, on=None):
    gpu.check(gpu.lib().nc_paged_plan(s.pool_ref, s.ref, on), "paged_plan")


def commit(gpu, s, finished=None, on=None):
    gpu.check(gpu.lib().nc_paged_commit(s.pool_ref, s.ref, P.ptr(finished), on), "paged_commit")


def assert_planned(s):
    sync()
    assert s.row_start.tolist() == s.want_rows
    assert s.kv_len.tolist() == [n + p for n, p in zip(s.new, s.past)]
    assert s.positions.tolist()[:s.max_tokens] == s.want_pos
    assert s.slots.tolist()[:s.max_tokens] == s.want_slots
    assert s.table.tolist() == s.want_table
    assert s.state.tolist()[:3] == [len(s.free_before), len(s.want_free), 0]


def gen(seed):
    return torch.Generator().manual_seed(seed)


CASES = {
    "one token, nothing cached": ([1], [0], 16, 0),
    "one token that opens a page": ([1], [16], 16, 0),
    "one token that fills a page": ([1], [15], 16, 0),
    "idle requests around": ([0, 3, 0, 0, 2, 0], [5, 0, 0, 33, 16, 64], 16, 3),
    "all idle": ([0, 0], [7, 0], 16, 4),
    "no rows at all": ([0], [0], 16, 0),
    "large pages": ([1000, 1, 1024], [1023, 1024, 0], 1024, 1),
    "chunks past one workgroup": ([700, 1, 0, 1500, 31], [1, 400, 9, 77, 5000], 32, 900),
}


@pytest.mark.parametrize("name", list(CASES))
def test_plan(gpu, name):
    new, past, page, pad = CASES[name]
    s = Step(new, past, page, gen(1), pad=pad)
    plan(gpu, s)
    assert_planned(s)
    plan(gpu, s)  # what it read it left: the same again
    assert_planned(s)


@pytest.mark.parametrize("n_req", [255, 256, 257, 1000, 4096])
def test_plan_many_requests(gpu, n_req):
    g = gen(n_req)
    new = torch.randint(0, 5, (n_req,), generator=g).tolist()
    past = torch.randint(0, 70, (n_req,), generator=g).tolist()
    s = Step(new, past, 16, g, pad=11)
    plan(gpu, s)
    assert_planned(s)


def test_last_page_is_taken_and_no_more(gpu):
    s = Step([17, 16], [0, 16], 16, gen(2), spare=0)
    assert len(s.want_free) == 0
    plan(gpu, s)
    assert_planned(s)


REFUSED = {
    "pages": (dict(new=[17, 16], past=[0, 16], spare=0), "NO_PAGES"),
    "kv": (dict(new=[2, 5], past=[3, 30], spare=9, max_kv=34), "TOO_LONG"),
    "rows": (dict(new=[4, 5], past=[3, 30], spare=9, pad=-1), "NO_ROWS"),
    "new": (dict(new=[2, 5], past=[3, 30], spare=9, max_new=4), "BAD_LEN"),
}


@pytest.mark.parametrize("why", list(REFUSED))
def test_plan_that_cannot_be_met_plans_nothing(gpu, why):
    kw, status = REFUSED[why]
    new, past = kw.pop("new"), kw.pop("past")
    spare = kw.pop("spare")
    s = Step(new, past, 16, gen(3), spare=spare, **kw)
    kw.update(new=new, past=past, spare=spare)
    if why == "pages":  # one page less than it takes
        s.state[0] -= 1
    free = s.state[0].item()
    plan(gpu, s)
    sync()
    assert s.state.tolist()[:3] == [free, free, getattr(gpu, "PLAN_" + status)]
    assert s.row_start.tolist() == [0] * (s.n_req + 1) and s.kv_len.tolist() == past
    assert s.positions.tolist() == [-1] * s.max_tokens and s.slots.tolist() == [-1] * s.max_tokens
    assert s.table.tolist() == s.table_before
    commit(gpu, s)
    sync()
    assert s.seq_len.tolist() == past and s.state[0].item() == free


@pytest.mark.parametrize("new,seq", [([-1, 2], [0, 0]), ([1, 2], [0, -5]), ([1, 2 ** 31 - 1], [0, 2 ** 31 - 1])])
def test_bad_lengths(gpu, new, seq):
    s = Step([1, 2], [0, 0], 16, gen(4), pad=5)
    s.new_len.copy_(ints(new))
    s.seq_len.copy_(ints(seq))
    plan(gpu, s)
    sync()
    assert s.state[2].item() & gpu.PLAN_BAD_LEN and s.row_start.tolist() == [0, 0, 0]
    assert s.slots.tolist() == [-1] * s.max_tokens and s.table.tolist() == s.table_before


def test_entry_that_is_no_page_gives_no_slot(gpu):
    s = Step([3, 3], [14, 3], 16, gen(5))
    s.table[0, 0] = s.n_pages  # the page of positions 14 and 15
    plan(gpu, s)
    sync()
    assert s.slots.tolist() == [-1, -1] + s.want_slots[2:]


def test_commit_takes_and_returns_pages(gpu):
    g = gen(6)
    s = Step([3, 20, 1, 0, 40], [14, 0, 31, 33, 8], 16, g)
    plan(gpu, s)
    finished = ints([0, 1, 0, 1, 5])
    commit(gpu, s, finished)
    sync()
    back, table = [], [list(t) for t in s.want_table]
    for r in (1, 3, 4):
        for j in range(P.up(s.new[r] + s.past[r], 16)):
            back.append(table[r][j])
            table[r][j] = -1
    free = s.want_free + back
    assert s.state.tolist()[:3] == [len(free), len(free), 0]
    assert s.free_pages.tolist()[:len(free)] == free
    assert s.table.tolist() == table
    assert s.seq_len.tolist() == [17, 0, 32, 0, 0] == s.kv_len.tolist()
    commit(gpu, s, finished)  # once more: nothing is left to return
    sync()
    assert s.state.tolist()[:2] == [len(free)] * 2 and s.seq_len.tolist() == [17, 0, 32, 0, 0]
    assert s.free_pages.tolist()[:len(free)] == free


@pytest.mark.parametrize("n_req", [63, 1025, 4096])
@pytest.mark.parametrize("share", [0.02, 0.5, 1.0])
def test_commit_many_requests(gpu, n_req, share):
    """Flags in more wavefronts and lots than one, pages in more than one load of a wavefront's."""
    g = gen(n_req)
    past = torch.randint(0, 60, (n_req,), generator=g).tolist()
    past[n_req // 2] = 1500
    s = Step([i % 3 for i in range(n_req)], past, 16, g)
    plan(gpu, s)
    done = (torch.rand(n_req, generator=g) < share).int().tolist()
    done[n_req // 2] = -1
    commit(gpu, s, ints(done))
    sync()
    free, table = list(s.want_free), [list(t) for t in s.want_table]
    for r in range(n_req):
        if done[r]:
            n = P.up(s.new[r] + s.past[r], 16)
            free += table[r][:n]
            table[r][:n] = [-1] * n
    assert s.state.tolist()[:3] == [len(free), len(free), 0]
    assert s.free_pages.tolist()[:len(free)] == free
    assert s.table.tolist() == table
    assert s.seq_len.tolist() == [0 if f else n + p for f, n, p in zip(done, s.new, past)]


def test_commit_passes_over_entries_that_are_no_page(gpu):
    s = Step([1], [79], 16, gen(7))
    plan(gpu, s)
    sync()
    s.table[0, 1], s.table[0, 3] = -1, s.n_pages + 4
    left = [s.want_table[0][j] for j in (0, 2, 4)]
    commit(gpu, s, ints([1]))
    sync()
    free = s.want_free + left
    assert s.state[0].item() == len(free) and s.free_pages.tolist()[:len(free)] == free


def test_pool_init(gpu):
    for n in (1, 5, 256, 1000):
        free, state = ints([-7] * n), ints([-7] * 4)
        pool = gpu.PagePool(free_pages=P.ptr(free), state=P.ptr(state), n_pages=n, page_size=16)
        gpu.check(gpu.lib().nc_page_pool_init(C.byref(pool), None), "page_pool_init")
        sync()
        assert free.tolist() == list(range(n - 1, -1, -1)) and state.tolist() == [n, n, 0, 0]


def test_steps_in_a_captured_graph(gpu):
    """Plan and commit captured once and replayed over many steps with changing lengths, against the host's allocator."""
    n_req, page, n_pages, n_tok = 6, 16, 40, 64
    g = gen(8)
    s = Step([1] * n_req, [0] * n_req, page, g, pad=n_tok - n_req, max_new=20, max_kv=100)
    s.n_pages = n_pages
    s.free_pages, s.state = ints([-1] * n_pages), ints([0] * 4)
    s.describe()
    finished = ints([0] * n_req)
    gpu.check(gpu.lib().nc_page_pool_init(s.pool_ref, None), "page_pool_init")
    sync()
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        plan(gpu, s, P.stream(torch.cuda.current_stream()))
        commit(gpu, s, finished, P.stream(torch.cuda.current_stream()))
    free, seq = list(range(n_pages - 1, -1, -1)), [0] * n_req
    table = [[-1] * s.max_pages for _ in range(n_req)]
    refused = 0
    for step in range(30):
        new = torch.randint(0, 12, (n_req,), generator=g).tolist()
        done = (torch.rand(n_req, generator=g) < 0.2).int().tolist()
        s.new_len.copy_(ints(new))
        finished.copy_(ints(done))
        graph.replay()
        sync()
        add = [P.up(a + n, page) - P.up(a, page) for a, n in zip(seq, new)]
        slots = []
        if sum(add) > len(free) or sum(new) > n_tok or any(a + n > 100 for a, n in zip(seq, new)):
            refused += 1
            new = [0] * n_req
        for r, n in enumerate(new):
            for i in range(seq[r], seq[r] + n):
                if i % page == 0:
                    table[r][i // page] = free.pop()
                slots.append(table[r][i // page] * page + i % page)
        for r in range(n_req):
            seq[r] += new[r]
            if done[r]:
                for j in range(P.up(seq[r], page)):
                    free.append(table[r][j])
                    table[r][j] = -1
                seq[r] = 0
        assert s.seq_len.tolist() == seq, step
        assert s.slots.tolist() == slots + [-1] * (n_tok - len(slots)), step
        assert s.state[0].item() == len(free) and s.free_pages.tolist()[:len(free)] == free, step
        assert s.table.tolist() == table, step
    assert 0 < refused < 25
