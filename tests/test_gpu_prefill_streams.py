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


@pytest.mark.parametrize("shared", [False, True])
def test_the_cached_attention_call(fd, shared):
    """Append, rotation and decode step in one call on another stream: grown lengths, rotated queries and results are its own."""
    B, Hq, Hkv, D, P = 6, 8, 2, 128, 16
    g = torch.Generator().manual_seed(5)
    lens = torch.tensor([40, 300, 5, 77, 1, 160], dtype=torch.int32, device=DEV)
    table = torch.randperm(B * 32, generator=g).int().view(B, 32).to(DEV)
    q, k, v = (torch.randn(B, 1, h, D, generator=g).to(BF16).to(DEV) for h in (Hq, Hkv, Hkv))
    pools = [torch.randn(B * 32 + 8, P, Hkv, D, generator=g).to(BF16).to(DEV) for _ in range(2)]
    tab = fd.layers._set_cos_sin_cache((1.0 / 10000.0 ** (torch.arange(0, D, 2, dtype=torch.float32) / D)).to(DEV), 1024)
    kw = dict(k=k, v=v, cache_seqlens=lens, block_table=table, cos_sin_cache=tab, position_ids=lens[:, None].long(),
              return_softmax_lse=True)
    if shared:
        kw["shared_prefix"] = (torch.tensor([100], dtype=torch.int32, device=DEV),
                               torch.arange(B * 32, B * 32 + 7, dtype=torch.int32, device=DEV).view(1, 7), None)
    got = []
    for on_side in (False, True, True):
        kw["cache_seqlens"] = lens.view(B, 1) if got else lens      # (as many numbers as sequences, in any shape)
        kc, vc = (p.clone() for p in pools)
        side = side_stream()
        if on_side:
            leave_writes_pending(B * 4, B * Hq * 4, B * Hq * D * 2, 1 << 20, 2 << 20)
        out, lse = fd.flash_attn_with_kvcache(q, kc, vc, **kw, **({"stream": side} if on_side else {}))
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        got.append((out, lse, kc, vc))
    for other in got[1:]:
        for a, b in zip(got[0], other):
            assert torch.equal(a, b)


@pytest.mark.parametrize("fuse", [False, True])
def test_decode_twins_on_a_stream(fd, fuse):
    pg = Paged([1, 400, 77, 1030], 8, 128, 16, BF16, seed=4)
    q = torch.randn(4, 32, 128, generator=torch.Generator().manual_seed(2)).to(BF16)
    args = (q.to(DEV), pg.k, pg.v, None, [1] * 4, pg.lens.to(DEV), pg.table.to(DEV), 0.09)
    want = oracle_prefill(q, pg.seq, [1] * 4, True, 0.09)
    need = fd.workspace_bytes(args[0], pg.k, args[6])
    for _ in range(3):
        lse = torch.empty(4, 32, device=DEV)
        side = side_stream()
        leave_writes_pending(q.numel() * 2, need, 4 * 4096)
        out = fd.gqa_fwd_batch_decode_aot(side, *args, lse_out=lse, fuse_combine=fuse)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        check(out, lse, *want, BF16, 1030, pg.vmax)
