"""Chunks that reach beyond the room of a sequence's block table: what fits is as if there were more room."""
import pytest
import torch

from test_gpu_prefill import BF16, DEV, Paged, check, plain_rows, starts
from test_gpu_serving import close, ids, make_block, positions

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv_split", [0, 1, 3])
@pytest.mark.parametrize("tokens,beyond", [(3, 1), (20, 10), (150, 100), (9, 40)])
def test_rows_keep_their_places(fd, tokens, beyond, kv_split):
    """kv_lens beyond the table: row i sees the keys j <= i + kv_len - n_q of those that the table holds."""
    Hq, Hkv, D, P, room = 8, 2, 128, 16, 256
    pg = Paged([room, 70], Hkv, D, P, BF16, seed=3, width_slack=0)
    ql = [tokens, 5]
    q = torch.randn(sum(ql), Hq, D, generator=torch.Generator().manual_seed(4)).to(BF16)
    lse = torch.empty(sum(ql), Hq, device=DEV)
    out = fd.gqa_fwd_batch_prefill(q.to(DEV), pg.k, pg.v, starts(ql).to(DEV), ids([room + beyond, 70]), pg.table.to(DEV), 0.09,
                                   lse_out=lse, kv_split=kv_split)
    ref = [plain_rows(q[:tokens].double(), pg.seq[0][0], pg.seq[1][0], [i + 1 + room + beyond - tokens for i in range(tokens)], 0.09),
           plain_rows(q[tokens:].double(), pg.seq[0][1], pg.seq[1][1], [i + 66 for i in range(5)], 0.09)]
    check(out, lse, *(torch.cat(x) for x in zip(*ref)), BF16, room, pg.vmax)


@pytest.mark.parametrize("kind", ["dense", "paged_fp8"])
@pytest.mark.parametrize("padded", [False, True])
def test_the_block_at_the_end_of_a_cache(fd, kind, padded):
    gen = torch.Generator().manual_seed(8)
    B, hidden, Hq, Hkv, D, L, first, T = 3, 256, 8, 2, 128, 64, 54, 20
    attn, tab = make_block(fd, hidden, Hq, Hkv, D, gen)
    x = torch.randn(B, first + T, hidden, generator=gen).to(BF16).to(DEV)
    real = [20, 12, 4]
    got = []
    for room in (L, 4 * L):
        kw = dict(num_layers=1, batch_size=B, max_length=room, kv_heads=Hkv, head_dim=D, dtype=BF16, world_size=1)
        cache = fd.layers.KV_Cache(**kw) if kind == "dense" else fd.layers.PagedKV_Cache(page_size=16, fp8=True, seed=4, **kw)
        attn.prefill(x[:, :first].contiguous(), positions(cache, first, B), tab, cache, 0)
        cache.inc_offset(first)
        got.append(attn.prefill(x[:, first:].contiguous(), positions(cache, T, B), tab, cache, 0,
                                q_lens=ids(real) if padded else None))
    for b in range(B):
        n = min(L - first, real[b] if padded else T)
        close(got[0][b, :n], got[1][b, :n])
    assert torch.isfinite(got[0].float()).all()
