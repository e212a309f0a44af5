"""NaN in queries, keys and scales of prompt attention and of the shared-prefix step: a row that meets one is NaN in output and
LSE, whatever the number of key ranges; all other rows are what they are without it (tolerances: see ``test_gpu_prefill``)."""
import math

import pytest
import torch

from test_gpu_prefill import BF16, DEV, FP16, Paged, check, oracle_prefill, oracle_shared, starts

pytestmark = pytest.mark.gpu


def check_rows(out, lse, ref, nan_rows, dtype, keys, vmax):
    """nan_rows [n, Hq]: rows that have to be NaN, output and LSE; the others agree with ref = (out, lse, magnitude)."""
    assert out.cpu()[nan_rows].isnan().all(), out.cpu()[nan_rows]
    assert lse.cpu()[nan_rows].isnan().all(), lse.cpu()[nan_rows]
    rest = ~nan_rows
    check(out.cpu()[rest], lse.cpu()[rest], *(t[rest] for t in ref), dtype, keys, vmax)


@pytest.mark.parametrize("kv_split", [1, 2, 4, 64])
@pytest.mark.parametrize("tokens,keys", [(3, 400), (150, 150), (40, 11)])        # key tiles, row tiles, rows that see nothing
@pytest.mark.parametrize("D,dtype", [(128, BF16), (64, FP16), (256, BF16)])
def test_a_nan_query_row(fd, kv_split, tokens, keys, D, dtype):
    g = torch.Generator().manual_seed(51)
    Hq, Hkv = 8, 2
    q = torch.randn(tokens, Hq, D, generator=g).to(dtype)
    k, v = (torch.randn(keys, Hkv, D, generator=g).to(dtype) for _ in range(2))
    ref = oracle_prefill(q, [[k.double()], [v.double()]], [tokens], True, D ** -0.5)
    nan_rows = torch.zeros(tokens, Hq, dtype=torch.bool)
    for i, h in ((tokens - 1, 5), (tokens // 2, 0), (0, 3)):
        q[i, h, (7 * i + h) % D] = math.nan
        nan_rows[i, h] = keys - tokens + i >= 0        # (a row that sees no key is 0 whatever it holds)
    lse = torch.empty(tokens, Hq, device=DEV)
    out = fd.gqa_fwd_batch_prefill(q.to(DEV), k.to(DEV), v.to(DEV), starts([tokens]).to(DEV), None, None, D ** -0.5,
                                   cu_seqlens_k=starts([keys]).to(DEV), lse_out=lse, kv_split=kv_split)
    check_rows(out, lse, ref, nan_rows, dtype, keys, 6.0)


@pytest.mark.parametrize("kv_split", [1, 2, 3])
@pytest.mark.parametrize("key", [0, 140, 299])
def test_a_nan_key_in_any_range(fd, kv_split, key):
    """All rows that see the key are NaN, also those whose other ranges are empty."""
    g = torch.Generator().manual_seed(52)
    n, Hq, Hkv, D = 300, 8, 2, 128
    q = torch.randn(n, Hq, D, generator=g).to(BF16)
    k, v = (torch.randn(n, Hkv, D, generator=g).to(BF16) for _ in range(2))
    ref = oracle_prefill(q, [[k.double()], [v.double()]], [n], True, D ** -0.5)
    k[key, 1, 77] = math.nan
    nan_rows = torch.zeros(n, Hq, dtype=torch.bool)
    nan_rows[key:, 4:] = True
    lse = torch.empty(n, Hq, device=DEV)
    out = fd.gqa_fwd_batch_prefill(q.to(DEV), k.to(DEV), v.to(DEV), starts([n]).to(DEV), None, None, D ** -0.5, lse_out=lse,
                                   kv_split=kv_split)
    check_rows(out, lse, ref, nan_rows, BF16, n, 6.0)


@pytest.mark.parametrize("Hq,Hkv,D,fp8", [(32, 8, 128, False), (8, 2, 64, True), (6, 1, 256, False)])
def test_a_nan_query_of_a_shared_prefix_step(fd, Hq, Hkv, D, fp8):
    """In a group, in a group without own keys, in no group, and one that sees no key at all."""
    members, pre_lens, own_lens = [4, 2], [333, 70], [17, 60, 0, 48, 5, 90, 33, 0]
    pg = Paged(own_lens + pre_lens, Hkv, D, 16, BF16, fp8=fp8, seed=D)
    B = len(own_lens)
    q = torch.randn(B, Hq, D, generator=torch.Generator().manual_seed(1)).to(BF16)
    own, pre = [s[:B] for s in pg.seq], [s[B:] for s in pg.seq]
    ref = oracle_shared(q, own, pre, members, D ** -0.5)
    nan_rows = torch.zeros(B, Hq, dtype=torch.bool)
    for b, h in ((0, 0), (2, Hq - 1), (5, 1), (6, 2), (7, 3)):
        q[b, h, 3] = math.nan
        nan_rows[b, h] = b != 7                        # (sequence 7: no group, no keys)
    lse = torch.empty(B, Hq, device=DEV)
    out = fd.gqa_fwd_batch_decode_shared_prefix(
        q.to(DEV), pg.k, pg.v, None, [1] * B, pg.lens[:B].to(DEV), pg.table[:B].to(DEV), pg.lens[B:].to(DEV),
        pg.table[B:].to(DEV), D ** -0.5, group_starts=starts(members).to(DEV), lse_out=lse, **pg.kw)
    check_rows(out, lse, ref, nan_rows, BF16, 500, pg.vmax)


@pytest.mark.parametrize("cap", [0.0, 8.0])
@pytest.mark.parametrize("tokens,kv_split", [(3, 1), (3, 4), (150, 1)])
def test_a_nan_scale(fd, cap, tokens, kv_split):
    """The softmax scale, and one KV head's scale of an fp8 cache; rows that see no key stay 0."""
    g = torch.Generator().manual_seed(53)
    Hq, Hkv, D = 8, 2, 128
    ql, kl = [tokens, tokens], [200, tokens - 2]            # (the second sequence: two rows without a key)
    pg = Paged(kl, Hkv, D, 16, BF16, fp8=True, seed=3)
    q = torch.randn(2 * tokens, Hq, D, generator=g).to(BF16)
    ref = oracle_prefill(q, pg.seq, ql, True, 0.09, cap)
    sees = torch.isfinite(ref[1])
    k_scale = pg.kw["k_scale"].clone()
    k_scale[1] = math.nan
    for scale, ks, nan_rows in ((math.nan, pg.kw["k_scale"], sees), (0.09, k_scale, sees & (torch.arange(Hq) >= 4))):
        lse = torch.empty(2 * tokens, Hq, device=DEV)
        out = fd.gqa_fwd_batch_prefill(q.to(DEV), pg.k, pg.v, starts(ql).to(DEV), pg.lens.to(DEV), pg.table.to(DEV), scale,
                                       cap, lse_out=lse, kv_split=kv_split, k_scale=ks, v_scale=pg.kw["v_scale"])
        check_rows(out, lse, ref, nan_rows, BF16, 200, pg.vmax)
