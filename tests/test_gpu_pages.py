"""Pages of a cache (copy, reserve, fork, free, compact) against a model of the same rules on the host: whole numbers and
bytes, so everything has to be equal."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
I32 = dict(dtype=torch.int32)


class Model:
    """Pools and tables on the CPU; every method is the documented rule, one page at a time."""

    def __init__(self, layers, pages, P, B, width, heads=2, dim=64, dtype=torch.bfloat16, seed=0, v_dim=None):
        g = torch.Generator().manual_seed(seed)
        size = torch.empty((), dtype=dtype).element_size()
        self.k, self.v = (torch.randint(0, 256, (layers, pages, P, heads, d * size), generator=g, dtype=torch.uint8)
                          .view(dtype) for d in (dim, v_dim or dim))
        self.table = torch.full((B, width), -1, **I32)
        self.lens = torch.zeros(B, **I32)
        self.refs = torch.zeros(pages, **I32)
        self.P = P

    def free_pages(self):
        return (self.refs == 0).nonzero()[:, 0].tolist()

    def copy(self, src, dst):
        for s, d in zip(src, dst):
            if 0 <= s < self.refs.numel() and 0 <= d < self.refs.numel():
                for pool in (self.k, self.v):
                    pool[:, d] = pool[:, s]

    def reserve(self, new):
        ok, free, used = [], self.free_pages(), 0
        for b in range(self.table.shape[0]):
            first, last = -(-int(self.lens[b]) // self.P), -(-(int(self.lens[b]) + new[b]) // self.P)
            if last > self.table.shape[1]:
                ok.append(0)
                continue
            missing = [j for j in range(first, last) if self.table[b, j] < 0]
            got = free[used:used + len(missing)]
            used += len(missing)
            ok.append(int(len(got) == len(missing)))
            if ok[-1]:
                for j, p in zip(missing, got):
                    self.table[b, j] = p
                    self.refs[p] = 1
        return ok

    def fork(self, parents, children):
        B = self.table.shape[0]
        ok, lens, table, free, plan = [], self.lens.clone(), self.table.clone(), self.free_pages(), []
        for i, (p, c) in enumerate(zip(parents, children)):
            good = 0 <= p < B and 0 <= c < B and p != c and lens[c] == 0 and table[c, 0] < 0 and c not in children[:i]
            if good and lens[p] % self.P:
                good = bool(free)
                plan.append((p, c, free.pop(0)) if good else None)
            elif good:
                plan.append((p, c, None))
            else:
                plan.append(None)
            ok.append(int(good))
        for job in plan:
            if job is None:
                continue
            p, c, page = job
            n = int(lens[p])
            whole, part = divmod(n, self.P)
            self.table[c, :whole] = table[p, :whole]
            self.refs[table[p, :whole].long()] += 1
            if page is not None:
                self.table[c, whole] = page
                self.refs[page] = 1
                for pool in (self.k, self.v):
                    pool[:, page, :part] = pool[:, int(table[p, whole]), :part]
            self.lens[c] = n
        return ok

    def free(self, rows):
        for r in rows:
            if 0 <= r < self.table.shape[0]:
                for j in range(self.table.shape[1]):
                    if self.table[r, j] >= 0:
                        self.refs[self.table[r, j]] -= 1
                        self.table[r, j] = -1
                self.lens[r] = 0

    def compact(self):
        n = int((self.refs > 0).sum())
        src = [p for p in range(n, self.refs.numel()) if self.refs[p] > 0]
        dst = [p for p in range(n) if self.refs[p] == 0]
        self.copy(src, dst)
        for s, d in zip(src, dst):
            self.table[self.table == s] = d
            self.refs[d], self.refs[s] = int(self.refs[s]), 0
        return n


class Pair:
    """The model and the GPU's tensors side by side."""

    def __init__(self, fd, *args, **kw):
        self.fd, self.m = fd, Model(*args, **kw)
        self.k, self.v, self.table, self.lens, self.refs = (t.to(DEV) for t in (self.m.k, self.m.v, self.m.table, self.m.lens,
                                                                                self.m.refs))

    def i32(self, x):
        return torch.tensor(x, **I32, device=DEV)

    def same(self, what=""):
        torch.cuda.synchronize()
        for name in ("table", "lens", "refs"):
            assert torch.equal(getattr(self, name).cpu(), getattr(self.m, name)), (what, name)
        for name in ("k", "v"):
            assert torch.equal(getattr(self, name).cpu().view(torch.uint8), getattr(self.m, name).view(torch.uint8)), (what, name)

    def reserve(self, new):
        each = new if isinstance(new, list) else [new] * self.table.shape[0]
        got = self.fd.paged_kv_reserve(self.table, self.lens, self.refs, self.i32(new) if isinstance(new, list) else new, self.m.P)
        want = self.m.reserve(each)
        assert got.tolist() == want
        self.same("reserve")
        return want

    def grow(self, new):
        """Reserve, and the lengths of the rows that got their pages go up."""
        each = new if isinstance(new, list) else [new] * self.table.shape[0]
        ok = self.reserve(new)
        step = torch.tensor([n if o else 0 for n, o in zip(each, ok)], **I32)
        self.m.lens += step
        self.lens += step.to(DEV)

    def fork(self, parents, children):
        got = self.fd.paged_kv_fork(self.k, self.v, self.table, self.lens, self.refs, self.i32(parents), self.i32(children))
        want = self.m.fork(parents, children)
        assert got.tolist() == want, (got.tolist(), want)
        self.same("fork")
        return want

    def free(self, rows):
        self.fd.paged_kv_free(self.table, self.lens, self.refs, self.i32(rows))
        self.m.free(rows)
        self.same("free")

    def compact(self):
        got = self.fd.paged_kv_compact(self.k, self.v, self.table, self.refs)
        want = self.m.compact()
        assert got.tolist() == [want]
        self.same("compact")


@pytest.mark.parametrize("layers,pages,P,heads,dim,dtype", [(1, 40, 16, 2, 64, torch.bfloat16), (3, 70, 1, 1, 64, torch.float32),
                                                            (2, 33, 7, 3, 64, torch.uint8), (2, 130, 64, 8, 128, torch.float16)])
def test_copy(fd, layers, pages, P, heads, dim, dtype):
    t = Pair(fd, layers, pages, P, 1, 1, heads, dim, dtype, v_dim=2 * dim)
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(1)).tolist()
    for n in (1, 3, pages // 2):
        src, dst = order[:n] + [-1, 2, 2 ** 31 - 1], order[pages - n:] + [3, pages, 4]
        if n == pages // 2:
            src, dst = src[:n], dst[:n]
        fd.paged_kv_copy(t.k, t.v, t.i32(src), t.i32(dst))
        t.m.copy(src, dst)
        t.same(n)
    fd.paged_kv_copy(t.k, t.v, t.i32([]), t.i32([]))
    fd.paged_kv_copy(t.k[0], t.v[0], t.i32([0]), t.i32([1]))       # pools of one layer
    t.m.k[0, 1], t.m.v[0, 1] = t.m.k[0, 0], t.m.v[0, 0]
    t.same("one layer")


def test_pools_that_are_slices(fd):
    """Layers and pages a distance apart: K and V as two halves of one allocation, tables as columns of a wider one."""
    g = torch.Generator().manual_seed(3)
    both = torch.randn(3, 20, 2, 16, 2, 64, generator=g).to(torch.bfloat16)
    wide = torch.full((4, 9), -1, **I32)
    dev, table = both.to(DEV), wide.to(DEV)
    lens, refs = torch.zeros(4, **I32, device=DEV), torch.zeros(20, **I32, device=DEV)
    fd.paged_kv_reserve(table[:, 2:6], lens, refs, torch.tensor([33, 0, 0, 5], **I32, device=DEV), 16)
    lens.copy_(torch.tensor([33, 0, 0, 5]))
    ok = fd.paged_kv_fork(dev[:, :, 0], dev[:, :, 1], table[:, 2:6], lens, refs, torch.tensor([0, 3], **I32, device=DEV),
                          torch.tensor([1, 2], **I32, device=DEV))
    assert ok.tolist() == [1, 1] and lens.tolist() == [33, 33, 5, 5]
    want = wide.clone()
    want[0, 2:5], want[3, 2], want[1, 2:5], want[2, 2] = torch.tensor([0, 1, 2]), 3, torch.tensor([0, 1, 4]), 5
    assert torch.equal(table.cpu(), want) and refs.tolist() == [2, 2, 1, 1, 1, 1] + [0] * 14
    both[:, 4, :, :1], both[:, 5, :, :5] = both[:, 2, :, :1], both[:, 3, :, :5]
    assert torch.equal(dev.cpu(), both)


def test_reserve(fd):
    t = Pair(fd, 1, 30, 16, 5, 6)
    t.grow([0, 1, 16, 17, 33])
    t.grow(0)
    t.grow(1)
    t.grow([15, 0, 0, 40, 1])
    assert t.reserve([97, 0, 0, 0, 0])[0] == 0 or int(t.lens[0]) + 97 <= 96      # wider than the table
    t.reserve([1, 90, 1, 1, 90])                                                 # the pool runs out on the way
    t.reserve([16] * 5)
    t.free([1, 3])
    t.grow([16, 96, 0, 3, 0])
    t.free([0, 1, 2, 3, 4])
    assert int(t.refs.sum()) == 0


@pytest.mark.parametrize("P", [1, 16, 48])
def test_fork_and_free(fd, P):
    t = Pair(fd, 2, 90 if P > 1 else 400, P, 12, 20 if P > 1 else 130, seed=P)
    t.grow([100, 0, 32, 0, 0, 5] + [0] * 6)
    assert t.fork([0, 0, 2, 5, 1], [1, 3, 4, 6, 7]) == [1, 1, 1, 1, 1]           # (an empty parent: an empty fork)
    # refused: a taken child, a child named twice, itself, out of range; a parent that is a child of the same call is empty
    assert t.fork([0, 2, 2, 8, 99, 0, -1, 9], [1, 8, 8, 8, 9, -3, 9, 10]) == [0, 1, 0, 0, 0, 0, 0, 1]
    t.grow([1] * 12)                                                            # both sides of a fork go on by themselves
    t.free([0, 0, 3, 77, -1, 11])
    t.free([0])
    t.fork([1, 1], [0, 3])
    t.free(list(range(12)))
    assert int(t.refs.sum()) == 0 and (t.table == -1).all()


def test_fork_without_a_free_page(fd):
    t = Pair(fd, 1, 8, 16, 6, 8)
    t.grow([100, 0, 0, 0, 0, 0])                                                # 7 pages, the last one part-filled
    assert t.fork([0, 0, 0], [1, 2, 3]) == [1, 0, 0]
    t.free([0])
    t.m.lens[1] = 96                                                            # full pages only: no page is needed
    t.lens[1] = 96
    assert t.fork([1, 1], [4, 5]) == [1, 1]


@pytest.mark.parametrize("pages,B,P", [(37, 6, 16), (5000, 40, 16), (9001, 70, 1)])
def test_compact(fd, pages, B, P):
    width = 130
    t = Pair(fd, 2, pages, P, B, width, heads=1, dim=64, seed=pages)
    g = torch.Generator().manual_seed(pages)
    t.compact()                                                                 # nothing lives
    for _ in range(3):
        t.grow(torch.randint(0, max(2, min(40 * P, pages * P // B // 2)), (B,), generator=g).tolist())
        t.free(torch.randperm(B, generator=g)[:B // 2].tolist())
        rows = [r for r in range(B) if t.m.lens[r] == 0 and t.m.table[r, 0] < 0]
        full = [r for r in range(B) if t.m.lens[r] > 0]
        if rows and full:
            t.fork([full[0]], [rows[0]])                                        # a shared page moves once
        t.compact()
        t.compact()                                                             # nothing moves
    t.free(list(range(B)))


def test_many_rows_and_a_large_pool(fd):
    """More rows than threads of the scan, and free pages several scan steps into the pool."""
    t = Pair(fd, 1, 20000, 1, 3000, 4, heads=1, dim=16)
    t.refs[:12345] = 7
    t.m.refs[:12345] = 7
    g = torch.Generator().manual_seed(1)
    t.grow(torch.randint(0, 5, (3000,), generator=g).tolist())
    t.fork(list(range(0, 1500)), list(range(1500, 3000)))


def test_refused_on_the_device_side_of_the_call(fd):
    k = torch.zeros(2, 8, 16, 2, 64, dtype=torch.bfloat16, device=DEV)
    table, lens, refs = (torch.zeros(s, **I32, device=DEV) for s in ((2, 4), (2,), (8,)))
    one = torch.zeros(1, **I32, device=DEV)
    for bad in (lambda: fd.paged_kv_copy(k[:, :, :, :1], k[:, :, :, :1], one, one),              # a page with gaps
                lambda: fd.paged_kv_copy(k, k[:, :4], one, one),                                   # different pages
                lambda: fd.paged_kv_copy(k, k, one.long(), one),
                lambda: fd.paged_kv_copy(k, k, one, torch.zeros(2, **I32, device=DEV)),
                lambda: fd.paged_kv_copy(k[..., :4].contiguous(), k[..., :4].contiguous()[..., :1], one, one),
                lambda: fd.paged_kv_reserve(table, lens, refs, -1, 16),
                lambda: fd.paged_kv_reserve(table.t(), lens, refs, 1, 16),
                lambda: fd.paged_kv_reserve(table, lens, refs, lens.long(), 16),
                lambda: fd.paged_kv_fork(k, k, table, lens, refs[:7], one, one),
                lambda: fd.paged_kv_fork(k, k, table, lens, refs, one, lens),
                lambda: fd.paged_kv_free(table, lens[:1], refs, one),
                lambda: fd.paged_kv_compact(k, k, table, refs.float())):
        with pytest.raises(RuntimeError):
            bad()
    torch.cuda.synchronize()


def test_pages_in_a_graph(fd):
    """Reserve, fork, free and compact captured once and replayed while the cache changes underneath."""
    t = Pair(fd, 2, 60, 16, 4, 12, seed=2)
    t.grow([40, 0, 25, 0])
    t.fork([0, 2], [1, 3])
    parents, children = t.i32([0, 2]), t.i32([1, 3])
    ok = t.i32([9, 9])
    granted = t.i32([9] * 4)
    live = t.i32([9])

    def step():
        fd.paged_kv_free(t.table, t.lens, t.refs, children)
        fd.paged_kv_fork(t.k, t.v, t.table, t.lens, t.refs, parents, children, ok_out=ok)
        fd.paged_kv_reserve(t.table, t.lens, t.refs, 9, 16, ok_out=granted)
        fd.paged_kv_compact(t.k, t.v, t.table, t.refs, live_out=live)

    def model():
        t.m.free([1, 3])
        a = t.m.fork([0, 2], [1, 3])
        b = t.m.reserve([9] * 4)
        return a, b, t.m.compact()

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    model()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    t.same("capture")
    for _ in range(4):
        g.replay()
        want = model()
        assert (ok.tolist(), granted.tolist(), int(live)) == want
        t.same("replay")
        t.lens += 5                       # the appends of a step, within what was reserved
        t.m.lens += 5
