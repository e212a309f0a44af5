"""Prompt attention (``gqa_fwd_batch_prefill``) and the shared-prefix decode step against a plain 64-bit softmax.

Tolerance of an output element, counted in roundings: with w the softmax weights, A = sum_j w_j |v_j| and h half a step of the
query's type, the kernel rounds every weight once (h A) and the result once (h |out|); the scores are sums of D products in 32
bits, wrong by at most D 2^-24 scale sum |q k| each, which for N(0, 1) inputs of D <= 256 stays below 2^-13 in the exponent and
twice that in a weight -- 2^-11 (A + |out|) covers it together with the sums over the keys.  fp16 weights below 2^-14 of the
reference point have an absolute error of 2^-25 each.  An LSE is a 32-bit logarithm of a 32-bit sum of such weights: 2^-12
absolute and 2^-22 relative.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, FP16, FP8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def plain_rows(q, k, v, visible, scale, cap=0.0):
    """q [n, Hq, D], k / v [m, Hkv, D] in float64; visible[i] keys are seen by row i -> out, lse, A."""
    n, Hq, D = q.shape
    m, Hkv, _ = k.shape
    out = torch.zeros(n, Hq, D, dtype=torch.float64)
    mag = torch.zeros_like(out)
    lse = torch.full((n, Hq), -math.inf, dtype=torch.float64)
    for h in range(Hq):
        x = (q[:, h] @ k[:, h // (Hq // Hkv)].t()) * scale
        if cap > 0:
            x = cap * torch.tanh(x / cap)
        see = torch.arange(m)[None] < torch.as_tensor(visible)[:, None]
        x = torch.where(see, x, -math.inf)
        lse[:, h] = torch.logsumexp(x, 1)
        w = torch.exp(x - torch.where(lse[:, h] > -math.inf, lse[:, h], 0.0)[:, None])
        vv = v[:, h // (Hq // Hkv)]
        for i in range(n) if not torch.isfinite(vv).all() else ():
            s = int(max(0, min(m, visible[i])))
            out[i, h], mag[i, h] = w[i, :s] @ vv[:s], w[i, :s] @ vv[:s].abs()
        if torch.isfinite(vv).all():
            out[:, h], mag[:, h] = w @ vv, w @ vv.abs()
    return out, lse, mag


def check(got, got_lse, out, lse, mag, dtype, keys, vmax):
    h = torch.finfo(dtype).eps / 2
    got, got_lse = got.double().cpu(), got_lse.double().cpu()
    tol = (h + 2.0 ** -11) * (mag + out.abs()) + (keys * 2.0 ** -25 * vmax if dtype == FP16 else 0.0) + 1e-30
    bad = (got - out).abs() > tol
    assert not bad.any(), (bad.nonzero()[:5].tolist(), (got - out)[bad][:5].tolist(), tol[bad][:5].tolist())
    assert torch.equal(torch.isfinite(got_lse), torch.isfinite(lse))
    fin = torch.isfinite(lse)
    assert ((got_lse - lse)[fin].abs() <= 2.0 ** -12 + 2.0 ** -22 * lse[fin].abs()).all(), (got_lse - lse)[fin].abs().max()
    assert (got_lse[~fin] == -math.inf).all()


class Paged:
    """Sequences in shuffled pages; what no sequence uses holds NaN (fp8: the NaN byte) or garbage table entries."""

    def __init__(self, lens, Hkv, D, P, dtype, fp8=False, seed=0, slack=3, poison=True, width_slack=2):
        g = torch.Generator().manual_seed(seed)
        need = [-(-n // P) for n in lens]
        pages = sum(need) + slack
        perm = torch.randperm(pages, generator=g)
        store = FP8 if fp8 else dtype
        src = [[torch.randn(n, Hkv, D, generator=g) for n in lens] for _ in range(2)]
        self.scales = [torch.rand(Hkv, generator=g) * 0.01 + 0.01 for _ in range(2)] if fp8 else [None, None]
        self.table = torch.randint(-9, pages + 9, (len(lens), max(need + [1]) + width_slack), generator=g, dtype=torch.int32)
        pools = [torch.full((pages * P, Hkv, D), math.nan if poison else 0.0).to(store) for _ in range(2)]
        self.seq = [[], []]
        at = 0
        for b, n in enumerate(lens):
            ids = perm[at:at + need[b]]
            at += need[b]
            self.table[b, :need[b]] = ids.int()
            slots = (ids[:, None] * P + torch.arange(P)[None]).reshape(-1)[:n]
            for i in range(2):
                x = src[i][b]
                if fp8:
                    x = (x / self.scales[i][None, :, None]).clamp(-448, 448)
                x = x.to(store)
                pools[i].view(torch.uint8 if fp8 else torch.int16)[slots] = x.view(torch.uint8 if fp8 else torch.int16)
                x = x.double()
                self.seq[i].append(x * self.scales[i].double()[None, :, None] if fp8 else x)
        self.k, self.v = (p.view(pages, P, Hkv, D).to(DEV) for p in pools)
        self.lens = torch.tensor(lens, dtype=torch.int32)
        self.vmax = max([1.0] + [float(x.abs().max()) for x in self.seq[1] if x.numel()])
        self.kw = dict(k_scale=self.scales[0].to(DEV), v_scale=self.scales[1].to(DEV)) if fp8 else {}


def starts(lens, first=0):
    return torch.tensor([first] + [first + sum(lens[:i + 1]) for i in range(len(lens))], dtype=torch.int32)


def visible_of(n, m, causal):
    return [i + 1 + m - n if causal else m for i in range(n)]


def oracle_prefill(q, seqs, ql, causal, scale, cap=0.0):
    outs, lses, mags = [], [], []
    at = 0
    for b, n in enumerate(ql):
        k, v = seqs[0][b], seqs[1][b]
        o, l, m = plain_rows(q[at:at + n].double(), k, v, visible_of(n, k.shape[0], causal), scale, cap)
        outs.append(o), lses.append(l), mags.append(m)
        at += n
    return torch.cat(outs), torch.cat(lses), torch.cat(mags)


# (query lengths, key lengths): nothing, one token, tile borders, fewer keys than queries, many short ones
LENGTHS = {
    "one": ([1], [1]),
    "square": ([5, 64, 129, 1, 0, 70], [5, 64, 129, 1, 0, 70]),
    "behind": ([3, 65, 0, 33, 1], [130, 65, 40, 300, 77]),
    "short_keys": ([40, 7, 3], [11, 0, 2]),
    "rows_128": ([128, 32], [128, 256]),
}
SHAPES = [(8, 2, 128), (32, 8, 128), (4, 4, 64), (6, 1, 256), (7, 1, 64), (3, 3, 256), (20, 1, 128)]


@pytest.mark.parametrize("lengths", list(LENGTHS))
@pytest.mark.parametrize("Hq,Hkv,D", SHAPES)
@pytest.mark.parametrize("kind", ["packed_bf16", "packed_fp16", "paged16_bf16", "paged1_fp16", "paged7_fp8"])
def test_against_plain(fd, lengths, Hq, Hkv, D, kind):
    ql, kl = LENGTHS[lengths]
    dtype = FP16 if "fp16" in kind else BF16
    g = torch.Generator().manual_seed(len(lengths) * 1000 + Hq + D)
    q = torch.randn(sum(ql), Hq, D, generator=g).to(dtype)
    for causal, cap, split in ((True, 0.0, 0), (False, 0.0, 1), (True, 0.0, 3), (True, 5.0, 0)):
        scale = D ** -0.5
        lse = torch.empty(sum(ql), Hq, device=DEV)
        if kind.startswith("packed"):
            seqs = [[torch.randn(n, Hkv, D, generator=g).to(dtype) for n in kl] for _ in range(2)]
            k, v = (torch.cat(s).to(DEV) for s in seqs)
            out = fd.gqa_fwd_batch_prefill(q.to(DEV), k, v, starts(ql).to(DEV), None, None, scale, cap, causal=causal,
                                           cu_seqlens_k=starts(kl).to(DEV), lse_out=lse, kv_split=split)
            seqs, vmax = [[x.double() for x in s] for s in seqs], 6.0
        else:
            P = 16 if "16_" in kind else 7 if "7_" in kind else 1
            pg = Paged(kl, Hkv, D, P, dtype, fp8="fp8" in kind, seed=Hq)
            out = fd.gqa_fwd_batch_prefill(q.to(DEV), pg.k, pg.v, starts(ql).to(DEV), pg.lens.to(DEV), pg.table.to(DEV),
                                           scale, cap, causal=causal, lse_out=lse, kv_split=split, **pg.kw)
            seqs, vmax = pg.seq, pg.vmax
        check(out, lse, *oracle_prefill(q, seqs, ql, causal, scale, cap), dtype, max(kl), vmax)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("fp8", [False, True])
def test_long_keys_many_tiles_and_split_ranges(fd, D, fp8):
    """Keys over many tiles; all split counts of one call agree with the plain result."""
    g = torch.Generator().manual_seed(D)
    ql, kl = [9, 260], [1500, 777]
    pg = Paged(kl, 2, D, 16, BF16, fp8=fp8, seed=D)
    q = torch.randn(sum(ql), 8, D, generator=g).to(BF16)
    ref = oracle_prefill(q, pg.seq, ql, True, D ** -0.5)
    for split in (0, 1, 2, 5, 64):
        lse = torch.empty(sum(ql), 8, device=DEV)
        out = fd.gqa_fwd_batch_prefill(q.to(DEV), pg.k, pg.v, starts(ql).to(DEV), pg.lens.to(DEV), pg.table.to(DEV),
                                       D ** -0.5, lse_out=lse, kv_split=split, **pg.kw)
        check(out, lse, *ref, BF16, max(kl), pg.vmax)


def test_many_sequences(fd):
    """More sequences than one pass of the tile search looks at, empty ones among them."""
    g = torch.Generator().manual_seed(3)
    ql = torch.randint(0, 6, (150,), generator=g).tolist()
    kl = [n + int(e) for n, e in zip(ql, torch.randint(0, 50, (150,), generator=g))]
    pg = Paged(kl, 1, 64, 16, BF16, seed=5)
    q = torch.randn(sum(ql), 4, 64, generator=g).to(BF16)
    lse = torch.empty(sum(ql), 4, device=DEV)
    out = fd.gqa_fwd_batch_prefill(q.to(DEV), pg.k, pg.v, starts(ql).to(DEV), pg.lens.to(DEV), pg.table.to(DEV), 0.125,
                                   lse_out=lse)
    check(out, lse, *oracle_prefill(q, pg.seq, ql, True, 0.125), BF16, max(kl), pg.vmax)


@pytest.mark.parametrize("split", [1, 4])
def test_rows_of_no_sequence_are_left_as_they_are(fd, split):
    """Rows before the first sequence, behind the last one and behind a padded sequence's own length."""
    g = torch.Generator().manual_seed(11)
    Hq, Hkv, D, T = 8, 2, 128, 3
    ql, kl, pad = [10, 10, 10], [50, 90, 300], [10, 4, 0]
    pg = Paged(kl, Hkv, D, 16, BF16, seed=2)
    q = torch.randn(T + sum(ql) + 5, Hq, D, generator=g).to(BF16)
    out = torch.full_like(q, 777.0).to(DEV)
    lse = torch.full((q.shape[0], Hq), 777.0, device=DEV)
    fd.gqa_fwd_batch_prefill(q.to(DEV), pg.k, pg.v, starts(ql, T).to(DEV), pg.lens.to(DEV), pg.table.to(DEV), 0.09,
                             q_lens=torch.tensor(pad, dtype=torch.int32, device=DEV), output=out, lse_out=lse,
                             kv_split=split)
    real = [T + 10 * b + i for b in range(3) for i in range(pad[b])]
    rest = [i for i in range(q.shape[0]) if i not in real]
    assert (out[rest] == 777.0).all() and (lse[rest] == 777.0).all()
    ref = oracle_prefill(q[real], pg.seq, pad, True, 0.09)
    check(out[real], lse[real], *ref, BF16, 300, pg.vmax)


@pytest.mark.parametrize("where", ["packed", "paged"])
def test_strided_operands(fd, where):
    """Queries, keys and values as slices of one projection, K and V interleaved in one pool, a strided output."""
    g = torch.Generator().manual_seed(21)
    Hq, Hkv, D, n = 8, 2, 64, 150
    qkv = torch.randn(n, Hq + 2 * Hkv, D, generator=g).to(BF16).to(DEV)
    q, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
    out = torch.zeros(n, Hq, 2 * D, dtype=BF16, device=DEV)[:, :, :D]
    lse = torch.empty(n, Hq, device=DEV)
    cu = torch.tensor([0, n], dtype=torch.int32, device=DEV)
    if where == "packed":
        fd.gqa_fwd_batch_prefill(q, k, v, cu, None, None, 0.125, output=out, lse_out=lse)
    else:
        P = 16
        both = torch.full((12, P, 2 * Hkv, D), math.nan, dtype=BF16, device=DEV)
        ids = torch.randperm(12, generator=g)[:10]
        slots = (ids[:, None] * P + torch.arange(P)).reshape(-1)[:n]
        both.view(-1, 2 * Hkv, D)[slots.to(DEV)] = qkv[:, Hq:]
        fd.gqa_fwd_batch_prefill(q, both[:, :, :Hkv], both[:, :, Hkv:], cu, torch.tensor([n], dtype=torch.int32, device=DEV),
                                 ids.int().view(1, -1).to(DEV), 0.125, output=out, lse_out=lse)
    ref = oracle_prefill(q.cpu(), [[k.cpu().double()], [v.cpu().double()]], [n], True, 0.125)
    check(out, lse, *ref, BF16, n, 6.0)


@pytest.mark.parametrize("scale,factor", [(-0.09, 1.0), (0.0, 1.0), (0.09, 30.0), (1e-4, 1.0)])
def test_scales_and_sharp_scores(fd, scale, factor):
    g = torch.Generator().manual_seed(31)
    n, m, Hq, Hkv, D = 40, 400, 4, 2, 128
    q = (torch.randn(n, Hq, D, generator=g) * factor).to(BF16)
    k, v = (torch.randn(m, Hkv, D, generator=g).to(BF16) for _ in range(2))
    lse = torch.empty(n, Hq, device=DEV)
    out = fd.gqa_fwd_batch_prefill(q.to(DEV), k.to(DEV), v.to(DEV), starts([n]).to(DEV), None, None, scale,
                                   cu_seqlens_k=starts([m]).to(DEV), lse_out=lse)
    ref, ref_lse, mag = oracle_prefill(q, [[k.double()], [v.double()]], [n], True, scale)
    # scores that are `factor` times larger are off by as many times more: D 2^-24 scale sum |q k|, sum |q k| < 2 D factor
    e = 4 * D * 2.0 ** -24 * abs(scale) * 2 * D * factor
    tol = (2.0 ** -8 + 2.0 ** -11 + e) * (mag + ref.abs())
    assert ((out.double().cpu() - ref).abs() <= tol).all()
    assert ((lse.double().cpu() - ref_lse).abs() <= 2.0 ** -12 + e).all()


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("D,kv_split", [(128, 1), (64, 2), (256, 1)])
def test_non_finite_values_reach_only_the_rows_that_see_them(fd, bad, D, kv_split):
    g = torch.Generator().manual_seed(41)
    n, Hq, Hkv = 150, 8, 2
    q = torch.randn(n, Hq, D, generator=g).to(BF16)
    k, v = (torch.randn(n, Hkv, D, generator=g).to(BF16) for _ in range(2))
    v[100, 1, 5] = bad       # one value of one KV head
    k[140, 0, 0] = math.nan  # a key: all of its row's weights
    lse = torch.empty(n, Hq, device=DEV)
    out = fd.gqa_fwd_batch_prefill(q.to(DEV), k.to(DEV), v.to(DEV), starts([n]).to(DEV), None, None, D ** -0.5, lse_out=lse,
                                   kv_split=kv_split).double().cpu()
    clean_v, clean_k = v.clone(), k.clone()
    clean_v[100, 1, 5] = 0.0
    clean_k[140, 0, 0] = 0.0
    ref, ref_lse, mag = oracle_prefill(q, [[clean_k.double()], [clean_v.double()]], [n], True, D ** -0.5)
    hit = torch.zeros(n, Hq, D, dtype=torch.bool)
    hit[100:, 4:, 5] = True
    assert ((out == bad) | (out.isnan() if math.isnan(bad) else torch.zeros_like(hit)))[100:, 4:, 5].all()
    hit[140:, :4] = True
    assert out[140:, :4].isnan().all()
    tol = (2.0 ** -8 + 2.0 ** -11) * (mag + ref.abs())
    assert ((out - ref).abs() <= tol)[~hit].all()


def test_what_lies_behind_a_sequence_is_not_read(fd):
    """The same call with NaN, infinities and zeros in the unused slots and pages gives the same bits."""
    ql, kl, got = [3, 70], [77, 129], []
    q = torch.randn(73, 8, 128, generator=torch.Generator().manual_seed(1)).to(BF16).to(DEV)
    for poison in (0.0, math.nan, math.inf):
        pg = Paged(kl, 2, 128, 16, BF16, seed=9, poison=False)
        used = torch.zeros(pg.k.shape[0] * 16, dtype=torch.bool)
        for b, n in enumerate(kl):
            used[(pg.table[b, :-(-n // 16)].long()[:, None] * 16 + torch.arange(16)).reshape(-1)[:n]] = True
        for pool in (pg.k, pg.v):
            pool.view(-1, 2, 128)[(~used).to(DEV)] = poison
        got.append(fd.gqa_fwd_batch_prefill(q, pg.k, pg.v, starts(ql).to(DEV), pg.lens.to(DEV), pg.table.to(DEV), 0.09))
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2]) and torch.isfinite(got[0]).all()


def test_wild_tables_and_offsets_stay_in_bounds(fd):
    """Page ids, lengths and offsets far outside their ranges are clamped: finite results, nothing else is promised."""
    q = torch.randn(40, 4, 128, device=DEV).to(BF16)
    pool = torch.randn(6, 16, 2, 128, device=DEV).to(BF16)
    i32 = dict(dtype=torch.int32, device=DEV)
    table = torch.tensor([[2 ** 31 - 1, -5, 3], [-2 ** 31, 7, 100]], **i32)
    for lens in ([48, 2 ** 31 - 1], [-7, 20]):
        for cu in ([0, 20, 40], [-100, 20, 2 ** 31 - 1], [30, 10, 40], [0, 0, 0]):
            for split in (1, 4):
                out = torch.zeros_like(q)
                fd.gqa_fwd_batch_prefill(q, pool, pool, torch.tensor(cu, **i32), torch.tensor(lens, **i32), table, 0.09,
                                         output=out, kv_split=split)
                packed = pool.view(-1, 2, 128)
                fd.gqa_fwd_batch_prefill(q, packed, packed, torch.tensor(cu, **i32), None, None, 0.09, output=out,
                                         cu_seqlens_k=torch.tensor([5, -9, 2 ** 31 - 1], **i32), kv_split=split)
                torch.cuda.synchronize()
                assert torch.isfinite(out.float()).all()


def test_single_tokens_agree_with_the_decode_step(fd):
    pg = Paged([1, 400, 77, 1030], 8, 128, 16, BF16, seed=4)
    q = torch.randn(4, 32, 128, generator=torch.Generator().manual_seed(2)).to(BF16)
    lse = torch.empty(4, 32, device=DEV)
    out = fd.gqa_fwd_batch_prefill(q.to(DEV), pg.k, pg.v, starts([1] * 4).to(DEV), pg.lens.to(DEV), pg.table.to(DEV), 0.09,
                                   lse_out=lse)
    ref = oracle_prefill(q, pg.seq, [1] * 4, True, 0.09)
    check(out, lse, *ref, BF16, 1030, pg.vmax)
    lse2 = torch.empty(4, 32, device=DEV)
    out2 = fd.gqa_fwd_batch_decode(q.to(DEV), pg.k, pg.v, None, [1] * 4, pg.lens.to(DEV), pg.table.to(DEV), 0.09, lse_out=lse2)
    check(out2, lse2, *ref, BF16, 1030, pg.vmax)


def test_pool_beyond_four_gib(fd):
    """Pages on both sides of 2^31 elements and 2^32 bytes of one pool (K and V share it)."""
    Hkv, D, P = 2, 128, 16
    pages = (2 ** 32 // 2) // (P * Hkv * D) + 600          # bytes beyond 2^32
    pool = torch.zeros(pages, P, Hkv, D, dtype=BF16, device=DEV)
    ids = [0, pages - 1, pages // 2, pages // 2 + 1, pages - 300]
    g = torch.Generator().manual_seed(6)
    data = torch.randn(len(ids), P, Hkv, D, generator=g).to(BF16)
    pool[torch.tensor(ids, device=DEV)] = data.to(DEV)
    q = torch.randn(20, 8, D, generator=g).to(BF16)
    n = len(ids) * P - 3
    seq = data.view(-1, Hkv, D)[:n].double()
    lse = torch.empty(20, 8, device=DEV)
    out = fd.gqa_fwd_batch_prefill(q.to(DEV), pool, pool, starts([20]).to(DEV),
                                   torch.tensor([n], dtype=torch.int32, device=DEV),
                                   torch.tensor([ids], dtype=torch.int32, device=DEV), 0.09, lse_out=lse)
    check(out, lse, *oracle_prefill(q, [[seq], [seq]], [20], True, 0.09), BF16, n, 6.0)
    del pool


def test_workspace_stream_and_repeatability(fd):
    pg = Paged([3000, 20], 2, 128, 16, BF16, seed=4)
    ql = [6, 2]
    q = torch.randn(8, 8, 128, generator=torch.Generator().manual_seed(2)).to(BF16).to(DEV)
    args = (q, pg.k, pg.v, starts(ql).to(DEV), pg.lens.to(DEV), pg.table.to(DEV))
    need = fd.prefill_workspace_bytes(*args)
    assert need > 0        # few rows over many keys: split ranges
    first = fd.gqa_fwd_batch_prefill(*args, 0.09)
    ws = torch.full((need,), 255, dtype=torch.uint8, device=DEV)     # (all ones: NaN)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    second = fd.gqa_fwd_batch_prefill(*args, 0.09, workspace=ws, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert torch.equal(first, second) and not (ws == 255).all()
    check(first, torch.zeros(8, 8) + oracle_prefill(q.cpu(), pg.seq, ql, True, 0.09)[1], *oracle_prefill(
        q.cpu(), pg.seq, ql, True, 0.09), BF16, 3000, pg.vmax)


# ------------------------------------------------------------------------------------------- shared prefixes

def oracle_shared(q, own, pre, members, scale, cap=0.0):
    """own / pre: [K sequences, V sequences]; members[g] sequences of group g, the rest of the batch in none."""
    outs, lses, mags = [], [], []
    group = [g for g, n in enumerate(members) for _ in range(n)]
    for b in range(q.shape[0]):
        kv = [torch.cat((pre[i][group[b]], own[i][b])) if b < len(group) else own[i][b] for i in range(2)]
        o, l, m = plain_rows(q[b:b + 1].double(), kv[0], kv[1], [kv[0].shape[0]], scale, cap)
        outs.append(o), lses.append(l), mags.append(m)
    return torch.cat(outs), torch.cat(lses), torch.cat(mags)


SHARED = {
    "one_group": ([5], [333], [17, 60, 1, 0, 48]),
    "groups": ([2, 0, 7, 1], [64, 900, 129, 1], [5, 70, 3, 0, 200, 16, 64, 33, 1, 90]),
    "no_prefix": ([3], [0], [5, 0, 70]),
    "outside": ([2, 1], [100, 20], [5, 6, 7, 8, 0]),
    "batch_66": ([40, 26], [300, 31], [(7 * i) % 45 for i in range(66)]),
}


@pytest.mark.parametrize("which", list(SHARED))
@pytest.mark.parametrize("Hq,Hkv,D", [(32, 8, 128), (8, 2, 64), (6, 1, 256), (20, 1, 128), (3, 3, 128)])
@pytest.mark.parametrize("kind", ["bf16_p16", "fp16_p1", "fp8_p7"])
def test_shared_prefix_against_plain(fd, which, Hq, Hkv, D, kind):
    members, pre_lens, own_lens = SHARED[which]
    dtype, fp8, P = (FP16 if "fp16" in kind else BF16), "fp8" in kind, int(kind.split("_p")[1])
    pg = Paged(own_lens + pre_lens, Hkv, D, P, dtype, fp8=fp8, seed=D + Hq)
    B = len(own_lens)
    q = torch.randn(B, Hq, D, generator=torch.Generator().manual_seed(1)).to(dtype)
    own, pre = [s[:B] for s in pg.seq], [s[B:] for s in pg.seq]
    for cap in (0.0, 4.0):
        lse = torch.empty(B, Hq, device=DEV)
        out = fd.gqa_fwd_batch_decode_shared_prefix(
            q.to(DEV), pg.k, pg.v, None, [1] * B, pg.lens[:B].to(DEV), pg.table[:B].to(DEV), pg.lens[B:].to(DEV),
            pg.table[B:].to(DEV), D ** -0.5, cap,
            group_starts=None if len(members) == 1 and members[0] == B else starts(members).to(DEV), lse_out=lse, **pg.kw)
        check(out, lse, *oracle_shared(q, own, pre, members, D ** -0.5, cap), dtype, 1000, pg.vmax)


def test_shared_prefix_long_and_a_workspace(fd):
    members, pre_lens = [9, 23], [5000, 2111]
    own_lens = [(37 * i) % 700 for i in range(32)]
    pg = Paged(own_lens + pre_lens, 2, 128, 16, BF16, seed=8)
    q = torch.randn(32, 8, 128, generator=torch.Generator().manual_seed(1)).to(BF16)
    own, pre = [s[:32] for s in pg.seq], [s[32:] for s in pg.seq]
    ref = oracle_shared(q, own, pre, members, 0.09)
    ws = torch.full((64 << 20,), 255, dtype=torch.uint8, device=DEV)
    for workspace in (None, ws):
        lse = torch.empty(32, 8, device=DEV)
        out = fd.gqa_fwd_batch_decode_shared_prefix(
            q.to(DEV), pg.k, pg.v, workspace, [1] * 32, pg.lens[:32].to(DEV), pg.table[:32].to(DEV), pg.lens[32:].to(DEV),
            pg.table[32:].to(DEV), 0.09, group_starts=starts(members).to(DEV), lse_out=lse, max_kv_len=700,
            max_prefix_len=5000)
        check(out, lse, *ref, BF16, 5700, pg.vmax)


def test_a_scale_that_changes_in_place_counts_as_it_is(fd):
    pg = Paged([40], 2, 64, 16, BF16, seed=1)
    q = torch.randn(1, 4, 64, generator=torch.Generator().manual_seed(3)).to(BF16)
    scale, cu, table, lens = torch.tensor(0.5), starts([1]).to(DEV), pg.table.to(DEV), pg.lens.to(DEV)
    for value in (0.5, 0.03125):
        scale.fill_(value)
        lse = torch.empty(1, 4, device=DEV)
        out = fd.gqa_fwd_batch_prefill(q.to(DEV), pg.k, pg.v, cu, lens, table, scale, lse_out=lse)
        check(out, lse, *oracle_prefill(q, pg.seq, [1], True, value), BF16, 40, pg.vmax)
        out = fd.gqa_fwd_batch_decode_shared_prefix(q.to(DEV), pg.k, pg.v, None, None, lens * 0, table, lens, table, scale,
                                                    lse_out=lse)
        check(out, lse, *oracle_prefill(q, pg.seq, [1], True, value), BF16, 40, pg.vmax)


@pytest.mark.parametrize("D,fp8", [(64, False), (128, True), (256, False)])
def test_shared_prefix_with_more_ranges_than_lanes(fd, D, fp8):
    own_lens, pre_lens = [130, 0, 700, 130, 1], [9000]     # one KV head: 64 ranges of the prefix and some of the own keys
    pg = Paged(own_lens + pre_lens, 1, D, 16, BF16, fp8=fp8, seed=D)
    q = torch.randn(5, 4, D, generator=torch.Generator().manual_seed(2)).to(BF16)
    own, pre = [s[:5] for s in pg.seq], [s[5:] for s in pg.seq]
    lse = torch.empty(5, 4, device=DEV)
    out = fd.gqa_fwd_batch_decode_shared_prefix(
        q.to(DEV), pg.k, pg.v, None, [1] * 5, pg.lens[:5].to(DEV), pg.table[:5].to(DEV), pg.lens[5:].to(DEV),
        pg.table[5:].to(DEV), 0.09, group_starts=torch.tensor([0, 4], dtype=torch.int32, device=DEV), lse_out=lse, **pg.kw)
    check(out, lse, *oracle_shared(q, own, pre, [4], 0.09), BF16, 9700, pg.vmax)


def test_graph_replays_agree_with_eager_calls(fd):
    """Two captured graphs (a prompt chunk, a shared-prefix step) replayed with new contents, eager work in between."""
    B, Hq, Hkv, D, P = 6, 8, 2, 128, 16
    own_lens, pre_lens = [40, 300, 5, 77, 1, 160], [1200]
    pg = Paged(own_lens + pre_lens, Hkv, D, P, BF16, seed=3, poison=False)
    table, lens = pg.table.to(DEV).clamp(0, pg.k.shape[0] - 1), pg.lens.to(DEV)
    q = torch.randn(12, Hq, D, device=DEV).to(BF16)
    cu = starts([2] * B).to(DEV)
    step_lens = lens[:B].clone()

    def chunk():
        return fd.gqa_fwd_batch_prefill(q, pg.k, pg.v, cu, step_lens, table[:B], 0.09, kv_split=3)

    def shared():
        return fd.gqa_fwd_batch_decode_shared_prefix(q[:B], pg.k, pg.v, None, [1] * B, step_lens, table[:B], lens[B:],
                                                     table[B:], 0.09)

    graphs = []
    for fn in (chunk, shared):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            fn()
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = fn()
        graphs.append((g, y, fn))
    for step in range(4):
        q.copy_(torch.randn(12, Hq, D, device=DEV))
        step_lens.copy_(torch.tensor([max(1, n - 3 * step) for n in own_lens], dtype=torch.int32))
        for g, y, fn in graphs:
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, fn()), step
            assert torch.isfinite(y.float()).all()
