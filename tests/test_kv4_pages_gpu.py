"""Pages handed out by qw3_page_slots: ids outside of any pool on the free stack or in the table refuse the whole call."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def _call(ops, dev, ctx, new, page, table, free, n_free, ws):
    """In place, as a program calls it; everything that the call may change."""
    d = dict(table=_i32(table, dev), free=_i32(free, dev), lens=_i32(ctx, dev), n_free=_i32([n_free], dev))
    cu, pos, slots, _, _ = ops.page_slots(d["lens"], _i32(new, dev), page, d["table"], d["free"], d["n_free"], sum(new) + 3, ws, kv_len=d["lens"], n_free_out=d["n_free"])
    return d, cu, pos, slots


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("n", [3, 700])
@pytest.mark.parametrize("where", ["first taken", "last taken", "table"])
@pytest.mark.parametrize("bad", [-1, -(2 ** 31), 2 ** 31 - 1, "limit"])
def test_a_bad_page_refuses_the_call(ops, cuda, page, n, where, bad):
    """Table, stack and lengths stay as they were, no slot is given, and the workspace reports it."""
    if bad == "limit":
        bad = (2 ** 31 - 1) // page       # the first id whose slots pass 31 bits
    ctx = [(7 * b) % (3 * page) for b in range(n)]
    new = [(5 * b) % 4 for b in range(n)]
    ctx[1], new[1] = page + 1, 2          # goes on in a page that it has
    ctx[2], new[2] = 2 * page, 1          # takes one
    have, need = [-(-c // page) for c in ctx], [-(-(c + x) // page) for c, x in zip(ctx, new)]
    taken, width = sum(need) - sum(have), max(need) + 1
    table = [[(3 * b + i) % 1000 for i in range(h)] + [-1] * (width - h) for b, h in enumerate(have)]
    free, n_free = list(range(1000, 1000 + taken + 5)), taken + 2
    if where == "table":
        table[1][1] = bad
    else:
        free[n_free - 1 if where == "first taken" else n_free - taken] = bad
    ws = ops.Workspace()
    d, cu, pos, slots = _call(ops, cuda, ctx, new, page, table, free, n_free, ws)
    with pytest.raises(ops.cabi.Qw3Error) as e:
        ws.check()
    assert e.value.status == ops.cabi.QW3_ERR_RANGE
    assert d["table"].tolist() == table and d["free"].tolist() == free and d["lens"].tolist() == ctx and d["n_free"].tolist() == [n_free]
    assert (cu == 0).all() and (pos == 0).all() and (slots == -1).all()
    ws.check()


@pytest.mark.parametrize("page", [16, 64])
def test_entries_that_no_token_needs_are_not_looked_at(ops, cuda, page):
    """Bad ids deeper in the stack, above its top, in entries of full blocks before, of idle requests and behind the last."""
    ctx, new = [page + 3, 2 * page, 5, 0], [1, page + 1, 0, 1]
    table = [[-1, 7, -1, -1], [-1, -5, -1, -1], [-1] * 4, [-1] * 4]
    free, n_free = [-1, 31, 32, 33, -1], 4
    ws = ops.Workspace()
    d, cu, pos, slots = _call(ops, cuda, ctx, new, page, table, free, n_free, ws)
    ws.check()
    assert d["table"].tolist() == [[-1, 7, -1, -1], [-1, -5, 33, 32], [-1] * 4, [31, -1, -1, -1]] and d["n_free"].tolist() == [1]
    assert cu.tolist() == [0, 1, page + 2, page + 2, page + 3] and d["lens"].tolist() == [c + x for c, x in zip(ctx, new)]
    assert slots.tolist() == [7 * page + 3] + [33 * page + i for i in range(page)] + [32 * page, 31 * page] + [-1] * 3
