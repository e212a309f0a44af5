"""Few query rows over many keys (tiles whose waves have keys of their own) and the sequences' own keys of a shared-prefix step:
values that are not finite, tables, offsets and lengths far outside their ranges, LSEs of a call in the caller's workspace."""
import math

import pytest
import torch

from test_gpu_prefill import BF16, DEV, FP16, FP8, Paged, check, oracle_prefill, oracle_shared, starts

pytestmark = pytest.mark.gpu


def check_hits(out, lse, ref, hit, bad, dtype, keys, vmax):
    """hit [n, Hq, D]: elements that see the value `bad`; everything else, and every LSE, is as without it."""
    out = out.cpu()
    got = out[hit].float()
    assert (got.isnan() if math.isnan(bad) else got == bad).all(), got[:8]
    o, l, mag = ref
    clean = torch.where(hit, o.to(out.dtype), out)
    check(clean, lse, torch.where(hit, clean.double(), o), l, mag, dtype, keys, vmax)


def put(pg, side, seq, token, head, dim, bad):
    """The value `bad` into K (0) or V (1) of a paged sequence; the oracle's copy gets 0."""
    P = pg.k.shape[1]
    pool = (pg.k, pg.v)[side]
    page = int(pg.table[seq, token // P])
    if pool.dtype == FP8:
        pool.view(torch.uint8)[page, token % P, head, dim] = 0x7f        # e4m3fn has NaN, no infinity
    else:
        pool[page, token % P, head, dim] = bad
    pg.seq[side][seq][token, head, dim] = 0.0


@pytest.mark.parametrize("kv_split", [1, 2, 4])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("D,kind", [(64, "bf16"), (128, "bf16"), (256, "bf16"), (64, "fp16"), (128, "fp16"), (64, "fp8"),
                                    (128, "fp8"), (256, "fp8")])
@pytest.mark.parametrize("tokens", [5, 100])             # key tiles, row tiles
def test_values_that_are_not_finite(fd, tokens, D, kind, causal, kv_split):
    """One V value that some rows, all rows and no rows of a sequence see; the last key, which fills up its block."""
    Hq, Hkv, P = 8, 2, 16
    dtype, fp8 = (FP16 if kind == "fp16" else BF16), kind == "fp8"
    for bad in (math.nan,) if fp8 else (math.inf, -math.inf, math.nan):
        for token in (397, 100, 399):
            pg = Paged([400, 150], Hkv, D, P, dtype, fp8=fp8, seed=D)
            put(pg, 1, 0, token, 1, 5, bad)
            q = torch.randn(2 * tokens, Hq, D, generator=torch.Generator().manual_seed(61)).to(dtype)
            lse = torch.empty(2 * tokens, Hq, device=DEV)
            out = fd.gqa_fwd_batch_prefill(q.to(DEV), pg.k, pg.v, starts([tokens] * 2).to(DEV), pg.lens.to(DEV),
                                           pg.table.to(DEV), D ** -0.5, causal=causal, lse_out=lse, kv_split=kv_split, **pg.kw)
            hit = torch.zeros(2 * tokens, Hq, D, dtype=torch.bool)
            first = max(0, token - 400 + tokens) if causal else 0         # row i sees the keys j <= i + 400 - tokens
            hit[first:tokens, 4:, 5] = True
            check_hits(out, lse, oracle_prefill(q, pg.seq, [tokens] * 2, causal, D ** -0.5), hit, bad, dtype, 400, pg.vmax)


@pytest.mark.parametrize("D,kind", [(64, "bf16"), (128, "fp16"), (256, "bf16"), (128, "fp8")])
@pytest.mark.parametrize("where", ["own_last", "own", "prefix_last", "prefix"])
def test_values_that_are_not_finite_in_a_shared_prefix_step(fd, D, kind, where):
    members, pre_lens, own_lens = [4, 2], [333, 70], [17, 60, 0, 48, 5, 90, 33]
    Hq, Hkv, B = 8, 2, 7
    dtype, fp8 = (FP16 if kind == "fp16" else BF16), kind == "fp8"
    for bad in (math.nan,) if fp8 else (math.inf, math.nan):
        pg = Paged(own_lens + pre_lens, Hkv, D, 16, dtype, fp8=fp8, seed=D)
        hit = torch.zeros(B, Hq, D, dtype=torch.bool)
        if where.startswith("own"):
            put(pg, 1, 1, 59 if where == "own_last" else 3, 0, 9, bad)
            hit[1, :4, 9] = True
        else:
            put(pg, 1, B, 332 if where == "prefix_last" else 100, 0, 9, bad)
            hit[:4, :4, 9] = True
        q = torch.randn(B, Hq, D, generator=torch.Generator().manual_seed(62)).to(dtype)
        own, pre = [s[:B] for s in pg.seq], [s[B:] for s in pg.seq]
        lse = torch.empty(B, Hq, device=DEV)
        out = fd.gqa_fwd_batch_decode_shared_prefix(
            q.to(DEV), pg.k, pg.v, None, [1] * B, pg.lens[:B].to(DEV), pg.table[:B].to(DEV), pg.lens[B:].to(DEV),
            pg.table[B:].to(DEV), D ** -0.5, group_starts=starts(members).to(DEV), lse_out=lse, **pg.kw)
        check_hits(out, lse, oracle_shared(q, own, pre, members, D ** -0.5), hit, bad, dtype, 500, pg.vmax)


@pytest.mark.parametrize("tokens", [5, 100])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_a_nan_byte_in_an_fp8_key(fd, D, tokens):
    """Rows that see the key are NaN."""
    Hq, Hkv = 8, 2
    pg = Paged([400], Hkv, D, 16, BF16, fp8=True, seed=D)
    put(pg, 0, 0, 398, 0, 7, math.nan)
    q = torch.randn(tokens, Hq, D, generator=torch.Generator().manual_seed(63)).to(BF16)
    lse = torch.empty(tokens, Hq, device=DEV)
    out = fd.gqa_fwd_batch_prefill(q.to(DEV), pg.k, pg.v, starts([tokens]).to(DEV), pg.lens.to(DEV), pg.table.to(DEV),
                                   D ** -0.5, lse_out=lse, **pg.kw).cpu()
    sees = torch.zeros(tokens, Hq, dtype=torch.bool)
    sees[tokens - 2:, :4] = True
    assert out[sees].isnan().all() and lse.cpu()[sees].isnan().all()
    check(out[~sees], lse.cpu()[~sees], *(t[~sees] for t in oracle_prefill(q, pg.seq, [tokens], True, D ** -0.5)), BF16, 400,
          pg.vmax)


# (every access that these values lead to is clamped: pages to the pool, table entries to the row's, rows to the query's)
WILD = [2 ** 31 - 1, -2 ** 31, -5, 7, 100]


def guarded(shape, dtype, fill):
    """A tensor in the middle of a larger one, and a check that what is around it has kept its value."""
    n = math.prod(shape)
    whole = torch.full((n + 8192,), fill, dtype=dtype, device=DEV)
    return whole[4096:4096 + n].view(shape), lambda: (whole[:4096] == fill).all() and (whole[4096 + n:] == fill).all()


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_wild_tables_and_offsets_of_few_rows(fd, D, fp8):
    i32 = dict(dtype=torch.int32, device=DEV)
    q = torch.randn(12, 4, D, device=DEV).to(BF16)
    pool = torch.randn(6, 16, 2, D, device=DEV).to(FP8 if fp8 else BF16)
    kw = dict(k_scale=torch.ones(2, device=DEV), v_scale=torch.ones(2, device=DEV)) if fp8 else {}
    table = torch.tensor([[2 ** 31 - 1, -5, 3], [-2 ** 31, 7, 100]], **i32)
    for lens in ([48, 2 ** 31 - 1], [-7, 20], [-2 ** 31, 1]):
        for cu in ([0, 6, 12], [-100, 6, 2 ** 31 - 1], [9, 3, 12], [0, 0, 0], [2 ** 31 - 1, -2 ** 31, 5]):
            for extra in (None, [2 ** 31 - 1, -3]):
                for split in (0, 1, 4):
                    out, whole = guarded(q.shape, BF16, 0.0)
                    fd.gqa_fwd_batch_prefill(q, pool, pool, torch.tensor(cu, **i32), torch.tensor(lens, **i32), table, 0.09,
                                             output=out, kv_split=split,
                                             q_lens=None if extra is None else torch.tensor(extra, **i32), **kw)
                    torch.cuda.synchronize()
                    assert whole() and torch.isfinite(out.float()).all()


@pytest.mark.parametrize("D,fp8", [(64, False), (128, True), (256, False)])
def test_wild_tables_offsets_and_lengths_of_a_shared_prefix_step(fd, D, fp8):
    """Sequences and groups that are in order agree with a call without the others."""
    i32 = dict(dtype=torch.int32, device=DEV)
    B = 5
    q = torch.randn(B, 4, D, device=DEV).to(BF16)
    pool = torch.randn(6, 16, 2, D, device=DEV).clamp(-2, 2).to(FP8 if fp8 else BF16)
    kw = dict(k_scale=torch.ones(2, device=DEV), v_scale=torch.ones(2, device=DEV)) if fp8 else {}
    good = torch.tensor([[0, 1, 2]] * B, **i32)
    own = torch.tensor([[0, 1, 2], WILD[:3], WILD[2:], WILD[1:4], [5, 5, 5]], **i32)
    for lens in ([40, 2 ** 31 - 1, -7, -2 ** 31, 30], [40, 48, 48, 0, 30]):
        for prefix_lens in ([33, 2 ** 31 - 1], [33, -9]):
            for groups in ([0, 2, 5], [0, 2, -1], [0, 2 ** 31 - 1, -2 ** 31], [3, 1, 4]):
                out, whole = guarded(q.shape, BF16, 0.0)
                fd.gqa_fwd_batch_decode_shared_prefix(
                    q, pool, pool, None, None, torch.tensor(lens, **i32), own, torch.tensor(prefix_lens, **i32),
                    torch.tensor([[3, 4, 5], WILD[:3]], **i32), 0.09, group_starts=torch.tensor(groups, **i32),
                    output_combine=out, **kw)
                torch.cuda.synchronize()
                assert whole()
                if groups == [0, 2, 5]:
                    assert torch.isfinite(out.float()).all()
                    alone = fd.gqa_fwd_batch_decode_shared_prefix(
                        q, pool, pool, None, None, torch.tensor([40, 0, 0, 0, 0], **i32), good, torch.tensor([33, 0], **i32),
                        torch.tensor([[3, 4, 5], [0, 0, 0]], **i32), 0.09, group_starts=torch.tensor(groups, **i32), **kw)
                    assert torch.equal(out[0], alone[0])


def test_the_callers_workspace_gives_the_same_lse(fd):
    """Rows over split key ranges: outputs and LSEs of a call with a workspace of its own and with the caller's."""
    pg = Paged([3000, 20], 2, 128, 16, BF16, seed=4)
    ql = [6, 2]
    q = torch.randn(8, 8, 128, generator=torch.Generator().manual_seed(2)).to(BF16)
    args = (q.to(DEV), pg.k, pg.v, starts(ql).to(DEV), pg.lens.to(DEV), pg.table.to(DEV))
    ws = torch.full((fd.prefill_workspace_bytes(*args),), 255, dtype=torch.uint8, device=DEV)
    got = []
    for workspace in (None, ws):
        lse = torch.full((8, 8), math.nan, device=DEV)
        out = fd.gqa_fwd_batch_prefill(*args, 0.09, workspace=workspace, lse_out=lse)
        check(out, lse, *oracle_prefill(q, pg.seq, ql, True, 0.09), BF16, 3000, pg.vmax)
        got.append((out, lse))
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1]) and not (ws == 255).all()


@pytest.mark.parametrize("tokens", [5, 100])
@pytest.mark.parametrize("cap", [30.0, 512.0, 4096.0])
def test_soft_caps_of_all_sizes(fd, cap, tokens):
    """A capped score, cap (1 - 2 / (1 + e^2y)), is off by a few roundings of numbers up to cap: 2^-22 cap, on top of what 32-bit
    products of large scores are off by (as in the test of sharp scores)."""
    g = torch.Generator().manual_seed(71)
    n, m, Hq, Hkv, D, scale, factor = tokens, 400, 4, 2, 128, 0.09, 20.0
    q = (torch.randn(n, Hq, D, generator=g) * factor).to(BF16)
    k, v = (torch.randn(m, Hkv, D, generator=g).to(BF16) for _ in range(2))
    lse = torch.empty(n, Hq, device=DEV)
    out = fd.gqa_fwd_batch_prefill(q.to(DEV), k.to(DEV), v.to(DEV), starts([n]).to(DEV), None, None, scale, cap,
                                   cu_seqlens_k=starts([m]).to(DEV), lse_out=lse)
    ref, ref_lse, mag = oracle_prefill(q, [[k.double()], [v.double()]], [n], True, scale, cap)
    e = 4 * D * 2.0 ** -24 * scale * 2 * D * factor + 2 * cap * 2.0 ** -22
    assert ((out.double().cpu() - ref).abs() <= (2.0 ** -8 + 2.0 ** -11 + e) * (mag + ref.abs())).all()
    assert ((lse.double().cpu() - ref_lse).abs() <= 2.0 ** -12 + e).all()


@pytest.mark.parametrize("batch", [65, 257, 1025, 2100])
@pytest.mark.parametrize("paged", [True, False])
def test_hundreds_and_thousands_of_sequences(fd, batch, paged):
    """Every row tile finds its sequence among all of them, empty ones and runs of empty ones included."""
    g = torch.Generator().manual_seed(batch)
    ql = torch.randint(0, 4, (batch,), generator=g).tolist()
    ql[batch // 3:batch // 2] = [0] * (batch // 2 - batch // 3)
    ql[-1] = 40
    kl = [n + int(e) for n, e in zip(ql, torch.randint(0, 30, (batch,), generator=g))]
    q = torch.randn(sum(ql), 2, 64, generator=g).to(BF16)
    lse = torch.empty(sum(ql), 2, device=DEV)
    if paged:
        pg = Paged(kl, 1, 64, 16, BF16, seed=5)
        seqs, vmax = pg.seq, pg.vmax
        out = fd.gqa_fwd_batch_prefill(q.to(DEV), pg.k, pg.v, starts(ql).to(DEV), pg.lens.to(DEV), pg.table.to(DEV), 0.125,
                                       lse_out=lse)
    else:
        seqs = [[torch.randn(n, 1, 64, generator=g).to(BF16) for n in kl] for _ in range(2)]
        k, v = (torch.cat(s).to(DEV) for s in seqs)
        seqs, vmax = [[x.double() for x in s] for s in seqs], 6.0
        out = fd.gqa_fwd_batch_prefill(q.to(DEV), k, v, starts(ql).to(DEV), None, None, 0.125,
                                       cu_seqlens_k=starts(kl).to(DEV), lse_out=lse)
    check(out, lse, *oracle_prefill(q, seqs, ql, True, 0.125), BF16, 100, vmax)
