"""Calls with ``stream=`` while the current stream is still busy with memory that has been given back to the allocator: what a
call allocates must not be that memory."""
import pytest
import torch

from test_gpu_pages import Pair
from test_gpu_prefill import BF16, DEV, Paged, check, oracle_prefill, oracle_shared, starts
from test_gpu_serving import make_block, positions

pytestmark = pytest.mark.gpu


def leave_writes_pending(*sizes):
    """Blocks of these sizes go back to the allocator while the current stream has yet to fill them with ones."""
    blocks = [torch.zeros(n, dtype=torch.uint8, device=DEV) for n in sizes for _ in range(3)]
    torch.cuda._sleep(100_000_000)
    for x in blocks:
        x.fill_(255)


def side_stream():
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    return side


def test_prefill_and_shared_prefix(fd):
    members, pre_lens, own_lens = [5, 3], [900, 70], [17, 60, 0, 48, 5, 90, 33, 1]
    pg = Paged(own_lens + pre_lens, 2, 128, 16, BF16, seed=4)
    g = torch.Generator().manual_seed(2)
    q, table, lens, groups = torch.randn(8, 8, 128, generator=g).to(BF16), pg.table.to(DEV), pg.lens.to(DEV), starts(members).to(DEV)
    qd, cu = q.to(DEV), starts([4, 4]).to(DEV)
    chunk_lens = pre_lens
    own, pre = [s[:8] for s in pg.seq], [s[8:] for s in pg.seq]
    want = oracle_prefill(q, pre, [4, 4], True, 0.09), oracle_shared(q, own, pre, members, 0.09)
    need = fd.prefill_workspace_bytes(qd, pg.k, pg.v, cu, lens[8:], table[8:], kv_split=8)
    for _ in range(3):
        lse = [torch.empty(8, 8, device=DEV) for _ in range(2)]
        side = side_stream()
        leave_writes_pending(need, q.numel() * 2, 4 * need)
        got = (fd.gqa_fwd_batch_prefill(qd, pg.k, pg.v, cu, lens[8:], table[8:], 0.09, lse_out=lse[0], kv_split=8, stream=side),
               fd.gqa_fwd_batch_decode_shared_prefix(qd, pg.k, pg.v, None, None, lens[:8], table[:8], lens[8:], table[8:], 0.09,
                                                     group_starts=groups, lse_out=lse[1], stream=side))
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        for out, l, ref in zip(got, lse, want):
            check(out, l, *ref, BF16, max(chunk_lens), pg.vmax)
        del got, out


def test_pages(fd):
    """Reserve, fork and compact: results, plans and the tables that follow from them."""
    for _ in range(3):
        t = Pair(fd, 2, 90, 16, 12, 20, seed=1)
        t.grow([100, 0, 32, 0, 0, 5] + [0] * 6)
        parents, children, new = t.i32([0, 0, 2, 5]), t.i32([1, 3, 4, 6]), t.i32([9] * 12)
        side = side_stream()
        leave_writes_pending(48, 12 * 4, 4, 16 + 90 * 12)
        forked = fd.paged_kv_fork(t.k, t.v, t.table, t.lens, t.refs, parents, children, stream=side)
        granted = fd.paged_kv_reserve(t.table, t.lens, t.refs, new, 16, stream=side)
        live = fd.paged_kv_compact(t.k, t.v, t.table, t.refs, stream=side)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        want = t.m.fork([0, 0, 2, 5], [1, 3, 4, 6]), t.m.reserve([9] * 12), t.m.compact()
        assert (forked.tolist(), granted.tolist(), int(live)) == want
        t.same()


def test_the_block_on_a_stream(fd):
    """A prompt and a decode step through the block on another stream while the current one is busy."""
    gen = torch.Generator().manual_seed(1)
    B, hidden, Hq, Hkv, D, T = 2, 256, 8, 2, 128, 37
    attn, tab = make_block(fd, hidden, Hq, Hkv, D, gen)
    x = torch.randn(B, T + 1, hidden, generator=gen).to(BF16).to(DEV)
    got = []
    for on_side in (False, True):
        cache = fd.layers.PagedKV_Cache(num_layers=1, batch_size=B, max_length=256, kv_heads=Hkv, head_dim=D, dtype=BF16,
                                        page_size=16, seed=4)
        pos = positions(cache, T, B), positions(cache, 1, B) + T
        first, last = x[:, :T].contiguous(), x[:, T:].contiguous()
        side = side_stream()
        kw = {"stream": side} if on_side else {}
        if on_side:
            leave_writes_pending(B * T * (Hq + 2 * Hkv) * D * 2, B * T * Hq * D * 2, B * T * hidden * 2, B * 4, B * hidden * 2)
        y = attn.prefill(first, pos[0], tab, cache, 0, **kw)
        with torch.cuda.stream(kw.get("stream", torch.cuda.current_stream())):
            cache.inc_offset(T)
        z = attn.fwd(last, pos[1], tab, cache, 0, **kw)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        got.append((y, z, cache.k_cache, cache.v_cache))
    for a, b in zip(*got):
        assert torch.equal(a, b)
