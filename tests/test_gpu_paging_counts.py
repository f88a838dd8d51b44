"""The page plan where a request's counts are no lengths (stale or garbage data, as large as an int): it is told, and the
requests around it are placed by the formula, number for number."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

LEFT = -77  # what the outputs hold before the call
MOST = 2**30 - 2**20


def formula(cached, new, table, free, T, P, width):
    """The plan of requests at rows 0, 1, .. (whole page table), in Python's integers, over the outputs' places alone."""
    told = 4 * any(v > MOST for v in cached + new)
    cached, new = ([min(max(v, 0), MOST) for v in x] for x in (cached, new))
    table, qsl, off, first = table.copy(), [0], 0, 0
    pos, loc, pt = np.zeros(T, np.int32), np.full(T, -1, np.int64), np.full((len(cached), width), LEFT, np.int32)
    for b, (c, n) in enumerate(zip(cached, new)):
        have, full = -(-c // P), -(-(c + n) // P)
        for j in range(have, min(full, table.shape[1])):
            if off + j - have < len(free):
                table[b, j] = free[off + j - have]
        slot = lambda key: (int(table[b, key // P]) * P + key % P  # noqa: E731
                            if key // P < table.shape[1] and (key // P < have or off + key // P - have < len(free)) else -1)
        for i in range(min(n, max(T - first, 0))):
            pos[first + i], loc[first + i] = c + i, slot(c + i) if c + i < width else -1
        for key in range(min(c + n, width)):
            pt[b, key] = max(slot(key), 0)
        told |= 4 * (full > table.shape[1]) | 8 * (c + n > width)
        off, first = off + full - have, first + n
        qsl.append(min(first, T))
    told |= (first > T) | 2 * (off > len(free))
    return qsl, [c + n for c, n in zip(cached, new)], pos, loc, [min(off, len(free)), told], table, pt


@pytest.mark.parametrize("P", [1, 4, 16, 1024])
@pytest.mark.parametrize("cached,new", [(2**31 - 1, 2**31 - 1), (2**30 - 1, 2**30 - 1), (2**31 - 1, 3), (MOST, 5), (MOST + 1, 0),
                                        (7, 2**31 - 1), (2**31 - 1, -2**31), (-2**31, 2**31 - 1)])
def test_a_request_of_garbage_counts(dev, P, cached, new):
    from bundles_amd.qwen36_layer import paging
    c, n, T, width = [5, cached, 9, 20], [3, new, 8, 1], 24, 40
    g = np.random.default_rng(P)
    table = g.permutation(4 * 48).reshape(4, 48).astype(np.int32)
    free = (1000 + g.permutation(60)).astype(np.int32)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    # (the list inside a larger allocation of a value of its own, which a place before or behind it would bring in)
    around = torch.full((4096,), 555, dtype=torch.int32, device=dev)
    around[2048:2108] = i32(free)
    tab, pt, plan = i32(table), torch.full((4, width), LEFT, dtype=torch.int32, device=dev), paging.PagePlan.alloc(4, T, dev)
    print(f"plan of {cached} + {new}, P={P}", flush=True)
    paging.plan_pages(i32(c), i32(n), tab, around[2048:2108], T, page_size=P, page_table=pt, plan=plan)
    torch.cuda.synchronize()
    qsl, lens, pos, loc, used, want_tab, want_pt = formula(c, n, table, free, T, P, width)
    assert plan.qsl.tolist() == qsl and plan.seqlens.tolist() == lens and plan.used.tolist() == used
    assert used[1] & paging.TABLE
    assert np.array_equal(plan.positions.cpu().numpy(), pos) and np.array_equal(plan.out_loc.cpu().numpy(), loc)
    assert np.array_equal(tab.cpu().numpy(), want_tab) and np.array_equal(pt.cpu().numpy(), want_pt)
