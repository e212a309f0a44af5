"""The cache's operators together, as a server runs them: pages are handed out, prompts go through the attention block, the
sequences are forked, decoded (also behind a shared prefix), freed and the pool is compacted -- with the block's results
against the same tokens in a cache that none of this happens to."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16 = torch.bfloat16


def make_block(fd, hidden, Hq, Hkv, D, gen, norm=True):
    mk = lambda *s, sc=0.06: (torch.randn(*s, generator=gen) * sc).to(BF16)  # noqa: E731
    attn = fd.layers.TP_Attn()
    attn.init_from_weights(mk(Hq * D, hidden), mk(Hkv * D, hidden), mk(Hkv * D, hidden), mk(hidden, Hq * D, sc=0.03), D)
    if norm:
        attn.q_norm_w, attn.k_norm_w = ((1 + mk(D, sc=0.1)).to(BF16).to(DEV) for _ in range(2))
        attn.q_norm_eps = attn.k_norm_eps = 1e-6
    tab = fd.layers._set_cos_sin_cache((1.0 / 10000.0 ** (torch.arange(0, D, 2, dtype=torch.float32) / D)).to(DEV), 1024)
    return attn, tab


def ids(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def positions(cache, n, B):
    return cache.kv_offset[:, None].long() + torch.arange(n, device=DEV)[None].expand(B, n)


def close(a, b):
    """Outputs of two orders of the same sums: each is off by a few roundings of the attention output (2^-8 relative to the
    magnitudes that are summed, here below 4 over `hidden` weights of 0.03) and of the result itself."""
    a, b = a.float(), b.float()
    assert torch.isfinite(a).all() and (a - b).abs().max().item() <= 2.0 ** -5, (a - b).abs().max().item()


@pytest.mark.parametrize("kind", ["dense", "paged", "paged_fp8", "managed", "managed_fp8"])
@pytest.mark.parametrize("D", [128, 64])
def test_prompt_in_chunks_equals_token_by_token(fd, kind, D):
    """A prompt through ``prefill`` in two chunks, the second padded, against the decode step token by token."""
    gen = torch.Generator().manual_seed(1)
    B, hidden, Hq, Hkv, L = 3, 256, 8, 2, 256
    attn, tab = make_block(fd, hidden, Hq, Hkv, D, gen)
    fp8 = kind.endswith("fp8")

    def cache():
        kw = dict(num_layers=2, batch_size=B, max_length=L, kv_heads=Hkv, head_dim=D, dtype=BF16, world_size=1)
        if kind == "dense":
            return fd.layers.KV_Cache(**kw)
        return fd.layers.PagedKV_Cache(page_size=16, fp8=fp8, seed=4, num_pages=60 if "managed" in kind else None, **kw)

    first, second = 37, [20, 1, 9]
    x = torch.randn(B, first + max(second), hidden, generator=gen).to(BF16).to(DEV)
    a, b = cache(), cache()
    managed = "managed" in kind
    if managed:
        assert a.reserve(first).tolist() == [1] * B
    got = [attn.prefill(x[:, :first], positions(a, first, B), tab, a, 1)]
    a.inc_offset(first)
    more = max(second)
    if managed:
        assert a.reserve(ids(second)).tolist() == [1] * B        # the padding has no pages: it lands in page 0
    got.append(attn.prefill(x[:, first:], positions(a, more, B), tab, a, 1, q_lens=ids(second)))
    a.inc_offset(ids(second))
    assert a.get_kv_len().tolist() == [first + n for n in second]
    for t in range(first + more):
        if managed:
            b.reserve(1)
        y = attn.fwd(x[:, t:t + 1], positions(b, 1, B), tab, b, 1)
        b.inc_offset()
        g = got[0][:, t:t + 1] if t < first else got[1][:, t - first:t - first + 1]
        for r in range(B):
            if t < first + second[r]:
                close(g[r], y[r])
    torch.cuda.synchronize()
    assert not a.k_cache[0].any()            # the other layer was never touched


def test_a_serving_run(fd):
    gen = torch.Generator().manual_seed(2)
    hidden, Hq, Hkv, D, L, B, P = 256, 8, 2, 128, 512, 6, 16
    attn, tab = make_block(fd, hidden, Hq, Hkv, D, gen)
    mk = lambda managed: fd.layers.PagedKV_Cache(num_layers=1, batch_size=B, max_length=L, kv_heads=Hkv, head_dim=D,  # noqa: E731
                                                 dtype=BF16, page_size=P, num_pages=120 if managed else None)
    a, b = mk(True), mk(False)               # pages handed out and moved / every row owns its pages
    prompt = torch.randn(2, 75, hidden, generator=gen).to(BF16).to(DEV)
    x = torch.zeros(B, 75, hidden, dtype=BF16, device=DEV)
    x[:2] = prompt
    n = ids([75, 60, 0, 0, 0, 0])
    assert a.reserve(n).tolist() == [1] * B
    ya = attn.prefill(x, positions(a, 75, B), tab, a, 0, q_lens=n)
    a.inc_offset(n)
    # the twin gets the same prompts in all six rows: 0, 1, and the forks 0, 0, 1, 0
    rows = [0, 1, 0, 0, 1, 0]
    yb = attn.prefill(x[rows], positions(b, 75, B), tab, b, 0, q_lens=n[rows].contiguous())
    b.inc_offset(n[rows])
    close(ya[0], yb[0]), close(ya[1, :60], yb[1, :60])
    assert a.fork(ids([0, 0, 1, 0]), ids([2, 3, 4, 5])).tolist() == [1, 1, 1, 1]
    assert a.kv_offset.tolist() == b.kv_offset.tolist() == [75, 60, 75, 75, 60, 75]
    shared = int((a.page_refs > 1).sum())
    assert shared == 75 // P + 60 // P       # the full pages of both prompts
    alive = list(range(B))
    for step in range(24):
        tok = torch.randn(B, 1, hidden, generator=gen).to(BF16).to(DEV)
        want = ids([1 if r in alive else 0 for r in range(B)])
        assert a.reserve(want).tolist() == [1] * B
        ya = attn.fwd(tok, positions(a, 1, B), tab, a, 0)
        yb = attn.fwd(tok, positions(b, 1, B), tab, b, 0)
        a.inc_offset(want), b.inc_offset(want)
        close(ya[alive], yb[alive])
        if step == 7:
            a.free(ids([0, 4]))              # a parent and a fork go; what the others share stays
            alive = [1, 2, 3, 5]
        if step == 12:
            live = int(a.compact())
            assert live == int((a.page_refs > 0).sum()) and (a.page_refs[live:] == 0).all() and int(a.page_refs[0]) == 1
    a.free(ids(list(range(B))))
    assert a.page_refs.tolist() == [1] + [0] * 119
    a.clear()
    assert int(a.page_refs.sum()) == 1 and (a.block_table == -1).all()


def test_decode_behind_a_shared_prefix(fd):
    """The prompt once in a row of its own, six sequences behind it; against caches that hold the prompt six times."""
    gen = torch.Generator().manual_seed(3)
    hidden, Hq, Hkv, D, L, B, P = 256, 8, 2, 128, 512, 6, 16
    attn, tab = make_block(fd, hidden, Hq, Hkv, D, gen)
    kw = dict(num_layers=1, max_length=L, kv_heads=Hkv, head_dim=D, dtype=BF16, page_size=P)
    a = fd.layers.PagedKV_Cache(batch_size=B + 1, num_pages=100, **kw)      # row 0: the prompt
    b = fd.layers.PagedKV_Cache(batch_size=B, **kw)
    n = 101
    prompt = torch.randn(1, n, hidden, generator=gen).to(BF16).to(DEV)
    assert a.reserve(ids([n] + [0] * B)).tolist() == [1] * (B + 1)
    x = torch.cat((prompt, torch.zeros(B, n, hidden, dtype=BF16, device=DEV)))
    attn.prefill(x, positions(a, n, B + 1), tab, a, 0, q_lens=ids([n] + [0] * B))
    a.inc_offset(ids([n] + [0] * B))
    attn.prefill(prompt.expand(B, n, hidden).contiguous(), positions(b, n, B), tab, b, 0)
    b.inc_offset(n)

    class Behind:                             # the rows behind the prompt as the block's cache
        k_scale = v_scale = None
        block_table = a.block_table[1:]

        def update_kv_cache(self, k, v, layer):
            return a.k_cache[layer], a.v_cache[layer], a.kv_offset[1:]

    for step in range(20):
        tok = torch.randn(B, 1, hidden, generator=gen).to(BF16).to(DEV)
        assert a.reserve(ids([0] + [1] * B)).tolist() == [1] * (B + 1)
        pos = (n + a.kv_offset[1:])[:, None].long()
        ya = attn.fwd(tok, pos, tab, Behind(), 0, shared_prefix=(a.kv_offset[:1], a.block_table[:1], None))
        yb = attn.fwd(tok, positions(b, 1, B), tab, b, 0)
        a.inc_offset(ids([0] + [1] * B)), b.inc_offset()
        close(ya, yb)


def test_only_a_managed_cache_hands_out_pages(fd):
    c = fd.layers.PagedKV_Cache(num_layers=1, batch_size=1, max_length=32, kv_heads=1, head_dim=64, dtype=BF16)
    for call in (lambda: c.reserve(1), lambda: c.fork(ids([0]), ids([0])), lambda: c.free(ids([0])), lambda: c.compact()):
        with pytest.raises(RuntimeError, match="num_pages"):
            call()
