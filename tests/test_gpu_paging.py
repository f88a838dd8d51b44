"""The page plan (q36_page_plan through paging.plan_pages) against a plain walk of the requests: row starts, key
counts, positions, slots, the extended block tables and the one-token page table, number for number; padded batches,
empty requests, pages that end inside a request's new tokens, and what does not fit."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

LEFT = -77  # what the outputs hold before the call


@pytest.fixture(scope="module")
def paging():
    from bundles_amd import _lib
    _lib.lib()
    from bundles_amd.qwen36_layer import paging
    return paging


def walk(cached, new, table, free, T, P, req, pt, whole):
    """The plan by hand; table and pt are changed in place."""
    cached, new = [max(c, 0) for c in cached], [max(n, 0) for n in new]
    B = len(cached)
    rows, width = table.shape
    qsl, used, total, bits = [0], 0, 0, 0
    pos, loc = np.zeros(T, np.int32), np.full(T, -1, np.int64)
    for b in range(B):
        r = b if req is None else int(req[b])
        ok = 0 <= r < rows
        n, have = cached[b] + new[b], -(-cached[b] // P)
        full = -(-n // P)
        pages = {}
        for j in range(full):
            if ok and j < width:
                if j < have:
                    pages[j] = int(table[r, j])
                elif used + j - have < len(free):
                    pages[j] = int(free[used + j - have])
                    table[r, j] = pages[j]
        pages = {j: p for j, p in pages.items() if 0 <= p < (2**31 - 1) // P}
        for i in range(new[b]):
            t, key = total + i, cached[b] + i
            if t < T:
                pos[t] = key
                fits = key // P in pages and (pt is None or key < pt.shape[1])
                loc[t] = pages[key // P] * P + key % P if fits else -1
        if pt is not None:
            for key in range(0 if whole else cached[b], min(n, pt.shape[1])):
                pt[b, key] = pages[key // P] * P + key % P if key // P in pages else 0
            bits |= 8 * (n > pt.shape[1])
        bits |= 4 * (not ok or full > width)
        used += full - have
        total += new[b]
        qsl.append(min(total, T))
    bits |= 1 * (total > T) | 2 * (used > len(free))
    return qsl, [c + n for c, n in zip(cached, new)], pos, loc, [min(used, len(free)), bits]


def make(cached, new, P, seed, spare=3, short=0, extra=2):
    g = np.random.default_rng(seed)
    full = [-(-(max(c, 0) + max(n, 0)) // P) for c, n in zip(cached, new)]
    have = [-(-max(c, 0) // P) for c in cached]
    B = len(cached)
    perm = g.permutation(sum(full) + 4).astype(np.int32)
    table = np.full((B + spare, max(full + [0]) + extra), LEFT, np.int32)
    req = g.permutation(B + spare)[:B].astype(np.int32)
    o = 0
    for b in range(B):
        table[req[b], :have[b]] = perm[o:o + have[b]]
        o += have[b]
    free = perm[o:]
    if short:
        free = free[:max(0, sum(full) - sum(have) - short)]
    return table, req, free


def run(paging, dev, cached, new, table, req, free, T, P, pt_width, whole):
    d = lambda v: torch.from_numpy(np.ascontiguousarray(v)).to(dev)  # noqa: E731
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    B = len(cached)
    tab, pt = d(table.copy()), None
    if pt_width:
        pt = torch.full((B, pt_width), LEFT, dtype=torch.int32, device=dev)
    plan = paging.PagePlan.alloc(B, T, dev)
    for t in (plan.qsl, plan.seqlens, plan.positions, plan.out_loc, plan.used):
        t.fill_(LEFT)
    got = paging.plan_pages(i32(cached), i32(new), tab, d(free), T, page_size=P, req=None if req is None else d(req),
                            page_table=pt, whole=whole, plan=plan)
    assert got is plan
    torch.cuda.synchronize()
    want_tab = table.copy()
    want_pt = np.full((B, pt_width), LEFT, np.int32) if pt_width else None
    qsl, lens, pos, loc, used = walk(cached, new, want_tab, free, T, P, req, want_pt, whole)
    assert plan.qsl.tolist() == qsl
    assert plan.seqlens.tolist() == lens
    assert plan.used.tolist() == used
    assert np.array_equal(plan.positions.cpu().numpy(), pos)
    assert np.array_equal(plan.out_loc.cpu().numpy(), loc)
    assert np.array_equal(tab.cpu().numpy(), want_tab)
    if pt_width:
        assert np.array_equal(pt.cpu().numpy(), want_pt)
    return plan


@pytest.mark.parametrize("P", [1, 2, 16, 64, 1024])
@pytest.mark.parametrize("whole", [True, False])
def test_plan_of_ragged_batches(paging, dev, P, whole):
    g = np.random.default_rng(P)
    for B, hi, n_hi in ((1, 1, 1), (1, 5000, 700), (7, 40, 1), (33, 300, 90), (301, 500, 9)):
        cached = g.integers(0, hi + 1, B).tolist()
        new = g.integers(0, n_hi + 1, B).tolist()
        print(f"plan P={P} whole={whole} B={B} up to {hi} + {n_hi}", flush=True)
        table, req, free = make(cached, new, P, B)
        width = max(c + n for c, n in zip(cached, new)) + 5
        for T in (sum(new), sum(new) + 13):
            run(paging, dev, cached, new, table, req, free, T, P, width, whole)
        run(paging, dev, cached, new, table, req, free, sum(new), P, 0, whole)


@pytest.mark.parametrize("P", [1, 16])
def test_page_borders_and_empty_requests(paging, dev, P):
    cached = [0, P, P - 1, 2 * P, 2 * P + 1, 0, 0, 5 * P, 3 * P - 1]
    new = [0, 1, 1, P, P - 1, P, 3 * P + 1, 0, 2]
    table, req, free = make(cached, new, P, 5)
    width = max(c + n for c, n in zip(cached, new))
    for whole in (True, False):
        run(paging, dev, cached, new, table, req, free, sum(new) + 3, P, width, whole)
        run(paging, dev, cached, new, table, req, free, sum(new), P, 0, whole)


def test_plan_without_request_rows(paging, dev):
    cached, new = [3, 0, 40], [2, 5, 1]
    table, req, free = make(cached, new, 4, 6, spare=0)
    straight = table[req]
    run(paging, dev, cached, new, straight, None, free, 8, 4, 50, True)


def test_no_new_tokens(paging, dev):
    table, req, free = make([9, 17], [0, 0], 16, 7)
    run(paging, dev, [9, 17], [0, 0], table, req, free, 0, 16, 20, True)
    run(paging, dev, [9, 17], [0, 0], table, req, free, 5, 16, 20, True)


def test_many_requests(paging, dev):
    g = np.random.default_rng(3)
    cached, new = g.integers(0, 20, 3001).tolist(), g.integers(0, 3, 3001).tolist()
    table, req, free = make(cached, new, 1, 8)
    run(paging, dev, cached, new, table, req, free, sum(new), 1, 23, True)


def test_what_does_not_fit_gets_no_slot(paging, dev):
    cached, new = [10, 0, 33, 7], [20, 9, 4, 30]
    P = 8
    table, req, free = make(cached, new, P, 9)
    width = max(c + n for c, n in zip(cached, new))
    p = run(paging, dev, cached, new, table, req, free, sum(new), P, width, True)
    assert p.used.tolist()[1] == 0
    # fewer rows than tokens, too few pages, a table and a page table that are too narrow, a row outside the table
    p = run(paging, dev, cached, new, table, req, free, 31, P, width, True)
    assert p.used.tolist()[1] == paging.TOKENS
    for short in (1, 3, 100):
        t2, r2, f2 = make(cached, new, P, 9, short=short)
        p = run(paging, dev, cached, new, t2, r2, f2, sum(new), P, width, False)
        assert p.used.tolist()[1] == paging.PAGES
    p = run(paging, dev, cached, new, table[:, :4].copy(), req, free, sum(new), P, width, True)
    assert p.used.tolist()[1] == paging.TABLE
    p = run(paging, dev, cached, new, table, req, free, sum(new), P, 31, True)
    assert p.used.tolist()[1] == paging.PAGE_TABLE
    for bad in (-1, table.shape[0], 2**31 - 1):
        r2 = req.copy()
        r2[2] = bad
        p = run(paging, dev, cached, new, table, r2, free, sum(new), P, width, True)
        assert p.used.tolist()[1] == paging.TABLE
    # counts and page numbers that are none
    t2, f2 = table.copy(), free.copy()
    t2[req[0], 0], t2[req[2], 1], f2[1] = -5, 2**31 - 1, -1
    run(paging, dev, [10, -3, 33, 7], [20, 9, -4, 30], t2, req, f2, sum(new), P, width, True)


def test_replayed_plan_follows_the_lengths(paging, dev):
    """One captured call serves the lengths that the buffers hold at each replay."""
    P, B, T, width = 4, 5, 40, 90
    rng = np.random.default_rng(1)
    table, req, free = make([60] * B, [20] * B, P, 2)
    d = lambda v: torch.from_numpy(np.ascontiguousarray(v)).to(dev)  # noqa: E731
    c, n, tab, fr, rq = (d(np.zeros(B, np.int32)), d(np.zeros(B, np.int32)), d(table), d(free), d(req))
    pt, plan = torch.zeros((B, width), dtype=torch.int32, device=dev), paging.PagePlan.alloc(B, T, dev)
    call = lambda: paging.plan_pages(c, n, tab, fr, T, page_size=P, req=rq, page_table=pt, plan=plan)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for _ in range(4):
        cached, new = rng.integers(0, 60, B).tolist(), rng.integers(0, 9, B).tolist()
        c.copy_(d(np.array(cached, np.int32)))
        n.copy_(d(np.array(new, np.int32)))
        tab.copy_(d(table))
        pt.fill_(LEFT)
        graph.replay()
        torch.cuda.synchronize()
        wt, wp = table.copy(), np.full((B, width), LEFT, np.int32)
        qsl, lens, pos, loc, used = walk(cached, new, wt, free, T, P, req, wp, True)
        assert plan.qsl.tolist() == qsl and plan.seqlens.tolist() == lens and plan.used.tolist() == used
        assert np.array_equal(plan.positions.cpu().numpy(), pos) and np.array_equal(plan.out_loc.cpu().numpy(), loc)
        assert np.array_equal(tab.cpu().numpy(), wt) and np.array_equal(pt.cpu().numpy(), wp)
