"""CPU-only checks of prompt attention, shared-prefix decode and the page operators: struct mirrors, argument validation of the
C entry points (nothing is launched without a GPU), launch plans, refusals of the wrappers."""
import ctypes
import os
import re

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FAKE = 0x10000


def _fields(name):
    with open(os.path.join(ROOT, "include", "flash_decode.h")) as f:
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), f.read(), re.S).group(1)
    out = []
    for decl in re.sub(r"/\*.*?\*/", "", body, flags=re.S).split(";"):
        if decl.strip():
            ctype, names = re.match(r"\s*(?:const\s+)?(\w+)\s*(.*)$", decl, re.S).groups()
            pointer = names.startswith("*")
            out += [(ctype, pointer or n.strip().startswith("*"), n.strip(" *\n")) for n in names.split(",")]
    return out


def test_structs_mirror_the_header(fd):
    L = fd._lib
    simple = {"int32_t": ctypes.c_int32, "int64_t": ctypes.c_int64, "float": ctypes.c_float, "fd_params": L.FdParams,
              "fd_decode_args": L.FdDecodeArgs}
    for cname, mirror in (("fd_prefill_args", L.FdPrefillArgs), ("fd_shared_args", L.FdSharedArgs),
                          ("fd_page_pool", L.FdPagePool), ("fd_page_tables", L.FdPageTables)):
        fields = _fields(cname)
        assert [f[2] for f in fields] == [n for n, _ in mirror._fields_], cname
        for (ctype, ptr, name), (_, pytype) in zip(fields, mirror._fields_):
            assert pytype is (ctypes.c_void_p if ptr else simple[ctype]), (cname, name)


def prefill_args(L, paged=True, batch=2, total_q=8, **params):
    a = L.FdPrefillArgs()
    a.q = a.k = a.v = a.out = a.cu_seqlens_q = FAKE
    if paged:
        a.block_table = a.kv_lens = FAKE
    else:
        a.cu_seqlens_k, a.total_k = FAKE, 100
    a.batch, a.total_q, a.causal, a.sm_scale = batch, total_q, 1, 0.1
    p = a.params
    p.q_heads, p.kv_heads, p.head_dim, p.page_size, p.num_pages, p.max_pages_per_seq = 32, 8, 128, 16, 64, 32
    p.q_dtype = p.kv_dtype = L.FD_BF16
    for name, value in params.items():
        setattr(p, name, value)
    a.stride_q_t, a.stride_q_h, a.stride_k_tok, a.stride_k_h, a.stride_v_tok, a.stride_v_h = 4096, 128, 1024, 128, 1024, 128
    a.stride_ot, a.stride_oh, a.stride_table_bs = 4096, 128, 32
    return a


def test_prefill_validates_before_it_launches(fd):
    L, lib = fd._lib, fd.load_library()

    def refused(a, code, text):
        need = lib.fd_prefill_workspace_bytes(ctypes.byref(a))
        if need > 0 and not a.workspace:
            a.workspace, a.workspace_bytes = FAKE, need
        assert lib.fd_prefill(None, ctypes.byref(a)) == code, lib.fd_last_error()
        assert text.encode() in lib.fd_last_error(), lib.fd_last_error()

    assert lib.fd_prefill(None, None) == -1 and lib.fd_prefill_workspace_bytes(None) == -1
    for params, code, text in (
            (dict(q_heads=30), -1, "multiple"), (dict(head_dim=96), -2, "head_dim"), (dict(v_head_dim=64), -2, "equal"),
            (dict(q_dtype=L.FD_F32), -2, "q_dtype"), (dict(kv_dtype=L.FD_F16), -2, "kv_dtype"),
            (dict(kv_dtype=L.FD_FP8_E4M3), -1, "k_scale"), (dict(num_splits=65), -1, "num_splits"),
            (dict(num_splits=-1), -1, "num_splits"), (dict(page_size=0), -1, "page_size"), (dict(num_pages=0), -1, "num_pages"),
            (dict(num_pages=1 << 20, page_size=1 << 12), -5, "2^31"),
            (dict(max_pages_per_seq=1 << 27), -5, "2^31")):
        refused(prefill_args(L, **params), code, text)
    refused(prefill_args(L, paged=False, kv_dtype=L.FD_FP8_E4M3), -2, "paged")
    refused(prefill_args(L, total_q=1 << 27), -5, "query rows")
    refused(prefill_args(L, batch=-1), -1, "batch")
    for field, value, code, text in (("q", None, -1, "NULL"), ("out", None, -1, "NULL"), ("cu_seqlens_q", None, -1, "offsets"),
                                     ("kv_lens", None, -1, "kv_lens"), ("q", FAKE + 8, -3, "aligned"),
                                     ("k", FAKE + 2, -3, "aligned"), ("stride_q_t", 4097, -3, "aligned"),
                                     ("stride_v_h", 132, -3, "aligned"), ("out", FAKE + 4, -3, "8-byte"),
                                     ("stride_oh", 130, -3, "8-byte")):
        a = prefill_args(L)
        setattr(a, field, value)
        refused(a, code, text)
    a = prefill_args(L, num_splits=4)
    need = lib.fd_prefill_workspace_bytes(ctypes.byref(a))
    assert need == 8 * 32 * 4 * (128 + 1) * 4
    for ws, size in ((None, need), (FAKE + 16, need), (FAKE, need - 1)):
        a.workspace, a.workspace_bytes = ws, size
        assert lib.fd_prefill(None, ctypes.byref(a)) == -1 and str(need).encode() in lib.fd_last_error()
    for empty in (prefill_args(L, batch=0), prefill_args(L, total_q=0)):
        assert lib.fd_prefill(None, ctypes.byref(empty)) == 0


def test_prefill_plan(fd):
    """Key ranges from sizes alone: none where the row tiles fill the chip, more the fewer there are, none for short keys."""
    L, lib = fd._lib, fd.load_library()

    def splits(total_q, batch, capacity, paged=True, **params):
        a = prefill_args(L, paged=paged, batch=batch, total_q=total_q, max_pages_per_seq=-(-capacity // 16), **params)
        a.total_k = capacity
        row = total_q * a.params.q_heads * (a.params.head_dim + 1) * 4
        need = lib.fd_prefill_workspace_bytes(ctypes.byref(a))
        assert need >= 0
        return round(need / row) if need else 1

    assert splits(16384, 1, 16384, paged=False) == 1 and splits(2048, 4, 32768) == 1
    assert splits(1, 1, 64) == 1 and splits(1, 1, 16384) > 8
    assert 1 < splits(256, 1, 16384) < splits(40, 1, 16384) <= 64
    assert splits(1, 1, 16384, max_kv_len=200) == 2 and splits(1, 1, 16384, max_kv_len=100) == 1
    assert splits(77, 1, 77, paged=False) == 1


def test_shared_prefix_validates_before_it_launches(fd):
    L, lib = fd._lib, fd.load_library()

    def args(**params):
        a = L.FdSharedArgs()
        s = a.step
        s.q = s.k_cache = s.v_cache = s.out = s.block_table = s.kv_lens = FAKE
        s.batch, s.sm_scale = 4, 0.1
        s.stride_q_bs, s.stride_q_h, s.stride_k_tok, s.stride_k_h, s.stride_v_tok, s.stride_v_h = 4096, 128, 1024, 128, 1024, 128
        s.stride_table_bs, s.stride_obs, s.stride_oh = 32, 4096, 128
        p = s.params
        p.q_heads, p.kv_heads, p.head_dim, p.page_size, p.num_pages, p.max_pages_per_seq = 32, 8, 128, 16, 64, 32
        p.q_dtype = p.kv_dtype = p.out_dtype = L.FD_BF16
        p.num_splits = -1
        for name, value in params.items():
            setattr(p, name, value)
        a.prefix_table = a.prefix_lens = a.group_starts = FAKE
        a.groups, a.prefix_max_pages, a.stride_prefix_bs = 1, 100, 100
        return a

    def refused(a, code, text, workspace=True):
        need = lib.fd_decode_shared_workspace_bytes(ctypes.byref(a))
        if workspace and need > 0:
            a.step.workspace, a.step.workspace_bytes = FAKE, need
        assert lib.fd_decode_shared(None, ctypes.byref(a)) == code, lib.fd_last_error()
        assert text.encode() in lib.fd_last_error(), lib.fd_last_error()

    assert lib.fd_decode_shared(None, None) == -1 and lib.fd_decode_shared_workspace_bytes(None) == -1
    refused(args(q_heads=30), -1, "multiple")
    refused(args(q_dtype=L.FD_F32, out_dtype=L.FD_F32), -2, "q_dtype")
    refused(args(out_dtype=L.FD_F32), -2, "query's type")
    refused(args(kv_dtype=L.FD_FP8_E4M3), -1, "k_scale")
    refused(args(v_head_dim=64), -2, "equal")
    refused(args(), -1, "workspace", workspace=False)
    for field, value, text in (("prefix_table", None, "NULL"), ("prefix_lens", None, "NULL"), ("groups", -1, "groups"),
                               ("prefix_max_pages", 0, "prefix_max_pages")):
        a = args()
        setattr(a, field, value)
        refused(a, -1, text)
    a = args()
    a.groups, a.group_starts = 2, None
    refused(a, -1, "offsets")
    for field, value in (("flags", 1), ("num_extra", 1), ("combine_mode", L.FD_COMBINE_SPLIT_LSE), ("seq_order", FAKE)):
        a = args()
        setattr(a.step, field, value)
        refused(a, -1, "FD_COMBINE_SPLIT")
    a = args()
    a.step.q = FAKE + 8
    refused(a, -3, "aligned")
    a = args()
    a.step.batch = 0
    assert lib.fd_decode_shared(None, ctypes.byref(a)) == 0 and lib.fd_decode_shared_workspace_bytes(ctypes.byref(a)) == 0


def test_pages_validate_before_they_launch(fd):
    L, lib = fd._lib, fd.load_library()

    def pool(**kw):
        p = L.FdPagePool()
        p.k_cache = p.v_cache = FAKE
        p.k_page_bytes = p.v_page_bytes = p.k_page_stride = p.v_page_stride = 4096
        p.k_layer_stride = p.v_layer_stride = 4096 * 8
        p.layers, p.num_pages, p.page_size = 2, 8, 16
        for name, value in kw.items():
            setattr(p, name, value)
        return ctypes.byref(p)

    def tables(**kw):
        t = L.FdPageTables()
        t.block_table = t.kv_lens = t.page_refs = FAKE
        t.stride_table_bs = t.max_pages_per_seq = 4
        t.batch = 3
        for name, value in kw.items():
            setattr(t, name, value)
        return ctypes.byref(t)

    ws = lib.fd_pages_workspace_bytes(8, 0)
    assert ws >= 8 * 12 and lib.fd_pages_workspace_bytes(8, 5) == 60 and lib.fd_pages_workspace_bytes(-1, 0) == -1
    for code, call in (
            (-1, lambda: lib.fd_pages_copy(None, None, FAKE, FAKE, 1)),
            (-1, lambda: lib.fd_pages_copy(None, pool(k_cache=None), FAKE, FAKE, 1)),
            (-1, lambda: lib.fd_pages_copy(None, pool(layers=0), FAKE, FAKE, 1)),
            (-5, lambda: lib.fd_pages_copy(None, pool(layers=40000), FAKE, FAKE, 1)),
            (-3, lambda: lib.fd_pages_copy(None, pool(k_page_bytes=4100, k_page_stride=8192), FAKE, FAKE, 1)),
            (-3, lambda: lib.fd_pages_copy(None, pool(v_cache=FAKE + 8), FAKE, FAKE, 1)),
            (-1, lambda: lib.fd_pages_copy(None, pool(v_page_stride=2048), FAKE, FAKE, 1)),
            (-1, lambda: lib.fd_pages_copy(None, pool(), None, FAKE, 1)),
            (-1, lambda: lib.fd_pages_copy(None, pool(), FAKE, FAKE, -1)),
            (-1, lambda: lib.fd_pages_reserve(None, None, 8, 16, None, 1, FAKE)),
            (-1, lambda: lib.fd_pages_reserve(None, tables(page_refs=None), 8, 16, None, 1, FAKE)),
            (-1, lambda: lib.fd_pages_reserve(None, tables(), 8, 0, None, 1, FAKE)),
            (-1, lambda: lib.fd_pages_reserve(None, tables(), 8, 16, None, -1, FAKE)),
            (-1, lambda: lib.fd_pages_reserve(None, tables(), 8, 16, None, 1, None)),
            (-5, lambda: lib.fd_pages_reserve(None, tables(batch=4097), 8, 16, None, 1, FAKE)),
            (-1, lambda: lib.fd_pages_fork(None, pool(), tables(batch=0), FAKE, FAKE, 1, FAKE, FAKE, 12)),
            (-1, lambda: lib.fd_pages_fork(None, pool(), tables(), None, FAKE, 1, FAKE, FAKE, 12)),
            (-1, lambda: lib.fd_pages_fork(None, pool(), tables(), FAKE, FAKE, 1, FAKE, None, 12)),
            (-1, lambda: lib.fd_pages_fork(None, pool(), tables(), FAKE, FAKE, 1, FAKE, FAKE, 11)),
            (-1, lambda: lib.fd_pages_free(None, tables(kv_lens=None), 8, FAKE, 1)),
            (-1, lambda: lib.fd_pages_free(None, tables(), 8, None, 1)),
            (-1, lambda: lib.fd_pages_compact(None, pool(), tables(), None, FAKE, ws)),
            (-1, lambda: lib.fd_pages_compact(None, pool(), tables(), FAKE, FAKE + 4, ws)),
            (-1, lambda: lib.fd_pages_compact(None, pool(), tables(), FAKE, FAKE, ws - 1))):
        assert call() == code and lib.fd_last_error()
    assert lib.fd_pages_copy(None, pool(), None, None, 0) == 0
    assert lib.fd_pages_fork(None, pool(), tables(), None, None, 0, None, None, 0) == 0
    assert lib.fd_pages_free(None, tables(), 8, None, 0) == 0


def test_wrappers_refuse_cpu_tensors_and_wrong_shapes(fd):
    q = torch.zeros(4, 8, 128, dtype=torch.bfloat16)
    kv = torch.zeros(6, 16, 2, 128, dtype=torch.bfloat16)
    i32 = torch.zeros(2, dtype=torch.int32)
    table = torch.zeros(1, 4, dtype=torch.int32)
    for call in (lambda: fd.gqa_fwd_batch_prefill(q, kv, kv, i32, i32[:1], table, 0.1),
                 lambda: fd.gqa_fwd_batch_prefill(q, q[:, :2], q[:, :2], i32, None, None, 0.1),
                 lambda: fd.prefill_workspace_bytes(q, kv, kv, i32, i32[:1], table),
                 lambda: fd.gqa_fwd_batch_decode_shared_prefix(q[:1], kv, kv, None, None, i32[:1], table, i32[:1], table, 0.1),
                 lambda: fd.paged_kv_copy(kv, kv, i32, i32),
                 lambda: fd.paged_kv_reserve(table, i32[:1], i32, 1, 16),
                 lambda: fd.paged_kv_fork(kv, kv, table, i32[:1], torch.zeros(6, dtype=torch.int32), i32, i32),
                 lambda: fd.paged_kv_free(table, i32[:1], i32, i32),
                 lambda: fd.paged_kv_compact(kv, kv, table, torch.zeros(6, dtype=torch.int32))):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()
    with pytest.raises(RuntimeError, match="q must be"):
        fd.gqa_fwd_batch_prefill(q[0], kv, kv, i32, i32[:1], table, 0.1)


class _OnGpu(torch.Tensor):
    """A CPU tensor that says it lives on a GPU: what the wrappers check before they touch the library."""
    is_cuda = True


def test_wrapper_checks_name_the_argument(fd):
    mk = lambda *s, dt=torch.bfloat16: torch.zeros(*s, dtype=dt).as_subclass(_OnGpu)  # noqa: E731
    i32 = lambda *s: mk(*s, dt=torch.int32)  # noqa: E731
    q, kv, cu, lens, table = mk(4, 8, 128), mk(6, 16, 2, 128), i32(3), i32(2), i32(2, 4)
    pre = fd.gqa_fwd_batch_prefill
    cases = [
        (lambda: pre(q, kv, kv, cu.long(), lens, table, 0.1), "cu_seqlens_q"),
        (lambda: pre(q, kv, kv, cu, lens[:1], table, 0.1), "kv_lens"),
        (lambda: pre(q, kv, kv, cu, None, table, 0.1), "kv_lens"),
        (lambda: pre(q, kv, kv, cu, lens, table[:1], 0.1), "block_table"),
        (lambda: pre(q, kv, kv, cu, lens, None, 0.1), "kv_lens"),
        (lambda: pre(q, kv, kv, cu, lens, table, 0.1, cu_seqlens_k=cu), "cu_seqlens_k"),
        (lambda: pre(q, kv, kv[:5], cu, lens, table, 0.1), "one shape"),
        (lambda: pre(q, kv, kv.float(), cu, lens, table, 0.1), "types"),
        (lambda: pre(q, kv[..., :64], kv[..., :64], cu, lens, table, 0.1), "head dims"),
        (lambda: pre(q, kv[:, :8], kv[:, :8], cu, lens, table, 0.1), "follow each other"),
        (lambda: pre(q, mk(6, 16, 3, 128), mk(6, 16, 3, 128), cu, lens, table, 0.1), "query heads"),
        (lambda: pre(q, kv, kv, cu, lens, table, 0.1, k_scale=mk(2, dt=torch.float32)), "together"),
        (lambda: pre(q, kv, kv, cu, lens, table, 0.1, k_scale=mk(3, dt=torch.float32), v_scale=mk(2, dt=torch.float32)), "scales"),
        (lambda: pre(q, kv, kv, cu, lens, table, 0.1, q_lens=i32(3)), "q_lens"),
        (lambda: pre(q, kv, kv, cu, lens, table, 0.1, output=mk(4, 8, 64)), "output"),
        (lambda: pre(q, kv, kv, cu, lens, table, 0.1, output=mk(4, 8, 128), lse_out=mk(4, 8)), "lse_out"),
        (lambda: pre(q, mk(9, 2, 128), mk(9, 2, 64), cu, None, None, 0.1), "packed"),
        (lambda: pre(q.clone().requires_grad_(), kv, kv, cu, lens, table, 0.1), "no backward"),
        (lambda: fd.gqa_fwd_batch_decode_shared_prefix(q, kv, kv, None, None, i32(4), i32(4, 2), lens, table, 0.1),
         "group_starts"),
        (lambda: fd.gqa_fwd_batch_decode_shared_prefix(q, kv, kv, None, None, i32(4), i32(4, 2), lens, table, 0.1,
                                                       group_starts=lens), "group_starts"),
        (lambda: fd.gqa_fwd_batch_decode_shared_prefix(q, kv, kv, None, None, i32(4), i32(4, 2), lens, i32(1, 2), 0.1),
         "prefix_lens"),
    ]
    for call, text in cases:
        with pytest.raises(RuntimeError, match=text):
            call()
