"""NaN in the decode step: a query head that meets one (in its query row, or in a key of its KV head) is NaN in output and LSE,
whatever the split count and the form of the merge; everything else is, bit for bit, what it is without it."""
import math

import pytest
import torch

from test_gpu_prefill import BF16, DEV, FP16, Paged

pytestmark = pytest.mark.gpu

# what leads through different merges: the library's plan, one split, few, many, the caller's partials, one fused launch, the
# scheduled variant, no allocation
FORMS = {
    "planned": {},
    "one": dict(kv_split=1, plan_splits=False),
    "four": dict(kv_split=4, plan_splits=False),
    "many": dict(kv_split=64, plan_splits=False),
    "many_general": dict(kv_split=80, plan_splits=False),
    "fused": dict(kv_split=4, fuse_combine=True),
    "no_alloc": dict(no_alloc=True),
    "two_waves": dict(kv_split=2, plan_splits=False, waves_per_block=2),
}


def call(fd, form, q, pg, lens, table, scale=0.09):
    B, Hq, D = q.shape
    kw = dict(pg.kw)
    out, lse = torch.empty(B, Hq, D, dtype=q.dtype, device=DEV), torch.empty(B, Hq, device=DEV)
    if form.startswith("partials"):
        mid = torch.empty(B, Hq, 32, D + 1, dtype=torch.float32 if form.endswith("fp32") else q.dtype, device=DEV)
        fd.gqa_fwd_batch_decode(q, pg.k, pg.v, None, None, lens, table, scale, 0.0, mid, out, 32, lse_out=lse, **kw)
    elif form == "scheduled":
        fd.gqa_fwd_batch_decode_persistent(q, pg.k, pg.v, None, None, lens, table, scale, output_combine=out, lse_out=lse, **kw)
    elif form == "column":
        both = fd.gqa_fwd_batch_decode_intra_rank(q, pg.k, pg.v, None, None, lens, table, scale, **kw)
        return both[..., :D].contiguous(), both[..., D].contiguous()
    else:
        fd.gqa_fwd_batch_decode(q, pg.k, pg.v, None, None, lens, table, scale, output_combine=out, lse_out=lse,
                                **FORMS[form], **kw)
    return out, lse


CASES = [((Hq, Hkv, D, kind), form)
         for Hq, Hkv, D, kind in ((32, 8, 128, "bf16"), (8, 2, 64, "fp16"), (8, 2, 256, "bf16"), (64, 2, 128, "bf16"),
                                  (32, 8, 128, "fp8"), (8, 2, 64, "fp8"), (8, 2, 256, "fp8"), (4, 2, 64, "fp32"))
         for form in (*FORMS, "partials_fp32", "partials", "scheduled", "column")
         if kind != "fp32" or form not in ("partials", "fused")]        # (partials in the query's type: in fp32 once)


@pytest.mark.parametrize("shape,form", CASES, ids=["-".join(map(str, shape)) + "-" + form for shape, form in CASES])
def test_a_nan_reaches_its_heads_and_no_others(fd, shape, form):
    Hq, Hkv, D, kind = shape
    dtype, fp8 = {"bf16": BF16, "fp16": FP16, "fp8": BF16, "fp32": torch.float32}[kind], kind == "fp8"
    lens = [400, 3000, 0, 37, 1, 2000]
    pg = Paged(lens, Hkv, D, 16, dtype, fp8=fp8, seed=D) if kind != "fp32" else None
    if pg is None:
        pg = Paged.__new__(Paged)
        g = torch.Generator().manual_seed(D)
        need = [-(-n // 16) for n in lens]
        pages = sum(need)
        pg.k, pg.v = (torch.randn(pages, 16, Hkv, D, generator=g).to(DEV) for _ in range(2))
        pg.table = torch.full((len(lens), max(need)), -1, dtype=torch.int32)
        for b, n in enumerate(need):
            pg.table[b, :n] = torch.arange(sum(need[:b]), sum(need[:b]) + n)
        pg.lens, pg.kw = torch.tensor(lens, dtype=torch.int32), {}
    q = torch.randn(len(lens), Hq, D, generator=torch.Generator().manual_seed(3)).to(dtype).to(DEV)
    table, lens_d = pg.table.to(DEV), pg.lens.to(DEV)
    clean = call(fd, form, q, pg, lens_d, table)
    assert torch.isfinite(clean[0]).all()
    nan_rows = torch.zeros(len(lens), Hq, dtype=torch.bool, device=DEV)
    for b, h in ((0, 0), (1, Hq - 1), (2, 1), (4, 1)):           # (sequence 2 holds no key: it stays 0 / -inf)
        q[b, h, 5] = math.nan
        nan_rows[b, h] = b != 2
    G = Hq // Hkv
    for b, token, h in ((1, 1999, 0), (3, 36, 1), (5, 0, 0)):
        slot = int(pg.table[b, token // 16]), token % 16, h, 7
        if fp8:
            pg.k.view(torch.uint8)[slot] = 0x7f
        else:
            pg.k[slot] = math.nan
        nan_rows[b, h * G:(h + 1) * G] = True
    out, lse = call(fd, form, q, pg, lens_d, table)
    torch.cuda.synchronize()
    assert out[nan_rows].isnan().all(), [i.tolist() for i in (nan_rows & ~out.isnan().all(-1)).nonzero()[:5]]
    assert lse[nan_rows].isnan().all(), [i.tolist() for i in (nan_rows & ~lse.isnan()).nonzero()[:5]]
    assert torch.equal(out[~nan_rows], clean[0][~nan_rows]) and torch.equal(lse[~nan_rows], clean[1][~nan_rows])


def test_a_nan_partial_of_another_rank(fd):
    """The merges over ranks and over further partials: NaN beside empty partials, and alone."""
    R, B, Hq, D = 3, 4, 8, 128
    parts = torch.randn(R, B, Hq, D + 1, device=DEV)
    lens = torch.tensor([[5, 0, 7, 0], [0, 0, 3, 1], [9, 4, 0, 0]], dtype=torch.int32, device=DEV)
    parts[0, 0, 1, D] = math.nan        # beside a valid partial
    parts[2, 1, 2, :] = math.nan        # the only valid one
    parts[1, 0, 3, :] = math.nan        # of a rank that holds nothing
    out, lse = torch.empty(B, Hq, D, dtype=BF16, device=DEV), torch.empty(B, Hq, device=DEV)
    fd.inter_rank_combine(parts, out, lens, lse_out=lse)
    want = torch.zeros(B, Hq, dtype=torch.bool, device=DEV)
    want[0, 1] = want[1, 2] = True
    assert torch.equal(out.isnan().all(-1), want) and torch.equal(out.isnan().any(-1), want) and torch.equal(lse.isnan(), want)
