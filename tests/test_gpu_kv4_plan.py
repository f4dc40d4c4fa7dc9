"""Plans whose page tables hold entries of no page: pages behind a window that
the caller has given back itself, and ids that are none of the cache's."""
import numpy as np
import pytest
import torch

import wohper_amd as wa
from test_gpu_kv4 import NONE, Plan, done

pytestmark = pytest.mark.gpu


def reclaim(p, rows, page_ids=NONE):
    """Takes pages away from requests' tables: onto the stack, `page_ids` in
    their place.  rows: request -> page indexes."""
    for b, which in rows.items():
        for i in which:
            p.stack.append(p.tables[b][i])
            p.tables[b][i] = page_ids
    stack = torch.tensor(np.asarray(p.stack, np.int64).astype(np.uint32).view(np.int32), device="cuda")
    p.d["free"][:len(p.stack)] = stack
    p.d["count"].fill_(len(p.stack))
    p.d["tables"].copy_(torch.tensor(np.asarray(p.tables, np.int64).astype(np.uint32).view(np.int32), device="cuda"))


def plain(p):
    """The plan in order, entries of no page passed over."""
    pages = lambda n: -(-n // p.page)  # noqa: E731
    tables, stack = [list(t) for t in p.tables], list(p.stack)
    for b, (o, n) in enumerate(zip(p.old, p.new)):
        stack += [i for i in tables[b][pages(n):pages(o)] if i < p.n_pages]
    seen = list(stack)
    slots = []
    for b, (o, n) in enumerate(zip(p.old, p.new)):
        for i in range(pages(o), pages(n)):
            tables[b][i] = stack.pop()
        slots += [tables[b][q // p.page] * p.page + q % p.page for q in range(o, n)]
    return tables, seen, len(stack), slots


def check(p):
    tables, seen, count, slots = plain(p)
    g = p.got()
    assert g["tables"] == tables and g["count_out"] == [count] and g["free_out"][:len(seen)] == seen
    assert g["slots"][:len(slots)] == slots and set(g["slots"][len(slots):p.max_tokens]) <= {NONE}


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("case", ["ends", "shrinks", "others_take_them", "all_none", "many"])
def test_pages_given_back_by_the_caller(ctx, case, in_place):
    """A request whose pages behind the window are gone ends or shrinks: what
    is left goes onto the stack, once."""
    if case == "many":
        rng = np.random.default_rng(1)
        old = rng.integers(1, 900, 1030).tolist()
        new = [0 if b % 3 == 0 else o + 40 if b % 3 == 1 else max(0, o - 100) for b, o in enumerate(old)]
        p = Plan(old, new, 4, in_place=in_place, extra=500)
        rows = {b: [i for i in range(-(-o // 4) - 9) if i >= 2] for b, o in enumerate(old) if b % 2 == 0}
    else:
        old, new = {"ends": ([1000, 50], [0, 51]), "shrinks": ([1000, 50], [300, 51]), "all_none": ([160, 3], [0, 3]),
                    "others_take_them": ([2600, 0, 64], [0, 1500, 900])}[case]
        p = Plan(old, new, 16, spare=0 if case == "others_take_them" else 3, in_place=in_place)
        rows = {0: range(10) if case == "all_none" else range(1, 55) if old[0] == 1000 else range(4, 150, 3)}
    reclaim(p, rows)
    torch.cuda.synchronize()
    ctx.kv_plan_async(p.s)
    done(ctx)
    check(p)


def test_more_table_entries_than_pages(ctx):
    """A long request of a small cache: most of its pages were given back."""
    p = Plan([3200, 0], [0, 100], 16, spare=0)
    reclaim(p, {0: range(190)})
    keep = p.tables[0][190:200]
    # ten pages are left of the request, and the cache has no others
    p.n_pages = p.s.n_pages = 10
    names = {v: i for i, v in enumerate(keep)}
    p.tables[0][190:200] = list(range(10))
    assert len(names) == 10
    p.stack = []
    p.d["tables"][0, 190:200] = torch.arange(10, device="cuda", dtype=torch.int32)
    p.d["count"].zero_()
    torch.cuda.synchronize()
    ctx.kv_plan_async(p.s)
    done(ctx)
    check(p)


def test_bad_pages_given_back_are_reported(ctx):
    """An id behind the cache does not get onto the stack."""
    p = Plan([100, 20], [0, 60], 16)
    reclaim(p, {0: [2]}, page_ids=p.n_pages)
    torch.cuda.synchronize()
    ctx.kv_plan_async(p.s)
    with pytest.raises(wa.DeepSeekV4KernelError) as e:
        ctx.synchronize()
    assert e.value.code == 10
    check(p)


def test_a_plan_that_only_entries_of_no_page_would_fit(ctx):
    """Entries of no page give nothing that others could take."""
    p = Plan([160, 0], [0, 100], 16, spare=0)
    p.d["count"].zero_()
    tables = [list(t) for t in p.tables]
    tables[0][:6] = [NONE] * 6  # four of the seven that are needed are left
    p.d["tables"].copy_(torch.tensor(np.asarray(tables, np.int64).astype(np.uint32).view(np.int32), device="cuda"))
    torch.cuda.synchronize()
    ctx.kv_plan_async(p.s)
    with pytest.raises(wa.DeepSeekV4KernelError) as e:
        ctx.synchronize()
    assert e.value.code == 11
    g = p.got()
    assert g["tables"] == tables and g["starts"] == [0] * 3 and g["count_out"] == [0] and set(g["slots"]) == {NONE}


@pytest.mark.parametrize("in_place", [False, True])
def test_more_pages_given_back_than_lds_holds(ctx, in_place):
    p = Plan([40000, 33, 70000, 0], [0, 34, 100, 50000], 4, in_place=in_place)
    torch.cuda.synchronize()
    ctx.kv_plan_async(p.s)
    done(ctx)
    p.check()
