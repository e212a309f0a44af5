"""Page operators on caches whose lengths and pages do not match, and at the limits of a call."""
import pytest
import torch

from test_gpu_pages import DEV, Pair

pytestmark = pytest.mark.gpu


def advance(t, rows, n):
    """Lengths go up without a word to the page operators."""
    for r in rows:
        t.lens[r] += n
        t.m.lens[r] += n


def test_a_length_without_pages_is_not_granted_more(fd):
    """A refusal that was not heeded and an idle row that was counted on: what their lengths count has no pages, so an append
    behind it would have a table with holes."""
    t = Pair(fd, 1, 6, 16, 4, 8)
    t.grow([48, 32, 0, 0])                                   # five of six pages
    assert t.reserve([16, 17, 0, 0]) == [1, 0, 0 + 1, 1]     # row 1 wants two pages, none is left
    advance(t, [0, 1, 2], 16)                                # row 1 and the idle row 2 go on all the same
    t.free([3])
    t.free([0])                                              # pages are free again
    before = t.table.clone(), t.refs.clone()
    ask = lambda new: fd.paged_kv_reserve(t.table, t.lens, t.refs, t.i32(new), 16).tolist()  # noqa: E731
    assert ask([0, 1, 1, 0]) == [1, 0, 0, 1]
    assert ask([0, 40, 17, 0]) == [1, 0, 0, 1]
    assert ask([0, 0, 0, 0]) == [1, 1, 1, 1]                 # nothing wanted, nothing to refuse
    assert torch.equal(t.table, before[0]) and torch.equal(t.refs, before[1])
    got = fd.paged_kv_fork(t.k, t.v, t.table, t.lens, t.refs, t.i32([1, 2]), t.i32([0, 3]))
    assert got.tolist() == [0, 0]                            # nor do they have all that a fork would share
    assert torch.equal(t.table, before[0]) and torch.equal(t.refs, before[1]) and t.lens.tolist() == [0, 48, 16, 0]
    t.free([1, 2])
    t.reserve([16, 0, 33, 0])                                # freed, they are rows like any other


def test_a_part_filled_page_that_is_missing(fd):
    """The next token would go into the page that the row lacks."""
    t = Pair(fd, 1, 8, 16, 2, 8)
    t.grow([16, 0])
    advance(t, [0, 1], 3)
    ok = fd.paged_kv_reserve(t.table, t.lens, t.refs, 1, 16)
    assert ok.tolist() == [0, 0] and t.table.tolist() == [[0] + [-1] * 7, [-1] * 8] and int(t.refs.sum()) == 1


def test_the_most_forks_of_a_call(fd):
    """Every child named twice, the second time in vain; many steps of the plan's scans."""
    n = 8192
    t = Pair(fd, 1, 3 * n, 16, n + 4, 2, heads=1, dim=16)
    for at, lens, pages in ((0, 17, [0, 1]), (1, 16, [2]), (2, 5, [3])):      # (more rows than a reserve takes)
        for lens_of, table, refs in ((t.lens, t.table, t.refs), (t.m.lens, t.m.table, t.m.refs)):
            lens_of[at] = lens
            for j, page in enumerate(pages):
                table[at, j], refs[page] = page, 1
    parents = [i % 4 for i in range(n)] + [0] * n
    children = [4 + (i * 5) % n for i in range(n)] + [4 + i for i in range(n)]
    assert len(parents) == 16384
    assert t.fork(parents, children) == [1] * n + [0] * n


def test_wild_tables_and_lists_stay_in_bounds(fd):
    """Page ids, lengths, counts and rows far outside their ranges: nothing around the tables and pools changes."""
    wild = [2 ** 31 - 1, -2 ** 31, -5, 100, 3, 0, 7, 99999]
    around = dict(dtype=torch.int32, device=DEV)
    whole = {name: torch.full((n + 512,), 123456, **around) for name, n in (("table", 32), ("lens", 4), ("refs", 8), ("ok", 4))}
    table, lens, refs, ok = (whole[n][256:256 + s] for n, s in (("table", 32), ("lens", 4), ("refs", 8), ("ok", 4)))
    table = table.view(4, 8)
    pool = torch.zeros(10, 2, 8, 16, 1, 64, device=DEV)       # (slice 4: K, slice 5: V, zeros around them)
    pool[4:6] = 1.0
    lists = torch.tensor([wild[:4], wild[4:]], **around)
    for round_ in range(4):
        table.copy_(torch.tensor([wild, wild[::-1], [-1] * 8, [-1] * 8], **around))
        lens.copy_(torch.tensor([[2 ** 31 - 1, -2 ** 31, 0, 40], [128, 129, -9, 5], [17, 33, 0, 0], [0, 0, 0, 0]][round_], **around))
        refs.copy_(torch.tensor([0, -4, 2 ** 31 - 1, 1, 0, 0, -2 ** 31, 3], **around))
        k, v = pool[4], pool[5]
        for rows in lists:
            fd.paged_kv_reserve(table, lens, refs, rows.abs().clamp(min=0), 16, ok_out=ok)
            fd.paged_kv_fork(k, v, table, lens, refs, rows, rows.flip(0).contiguous(), ok_out=ok)
            fd.paged_kv_copy(k, v, rows, rows.flip(0).contiguous())
            fd.paged_kv_compact(k, v, table, refs)
            fd.paged_kv_free(table, lens, refs, rows)
            torch.cuda.synchronize()
    for name, t in whole.items():
        assert (t[:256] == 123456).all() and (t[-256:] == 123456).all(), name
    assert not pool[:4].any() and not pool[6:].any() and (pool[4:6] == 1.0).all()
