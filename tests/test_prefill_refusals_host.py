"""CPU-only: calls that prompt attention, shared-prefix decode and the page operators refuse, and that nothing is done before."""
import pytest
import torch


def test_shared_prefix_keywords_are_refused_before_the_append(fd):
    q = torch.zeros(2, 1, 8, 128, dtype=torch.bfloat16)
    kv = torch.zeros(6, 16, 2, 128, dtype=torch.bfloat16)
    new = torch.zeros(2, 1, 2, 128, dtype=torch.bfloat16)
    i32 = torch.zeros(2, dtype=torch.int32)
    table = torch.zeros(2, 4, dtype=torch.int32)

    def call(**kw):
        return fd.flash_attn_with_kvcache(q, kv, kv, k=new, v=new, cache_seqlens=i32, block_table=table,
                                          shared_prefix=(i32[:1], table[:1], None), **kw)

    with pytest.raises(NotImplementedError, match="num_splits"):
        call(num_splits=4)
    for name in ("auto_order", "waves_per_block", "workspace", "no_such_keyword"):
        with pytest.raises(TypeError, match=name):
            call(**{name: 1})
    with pytest.raises(RuntimeError, match="no CPU path"):       # what is allowed goes on to the append
        call(max_kv_len=64, max_prefix_len=64)


def test_prefill_keywords_are_refused_before_the_append(fd):
    attn = fd.layers.TP_Attn()
    for name in ("output", "cu_seqlens_k", "k_scale", "no_such_keyword"):
        with pytest.raises(TypeError, match="unexpected keyword " + name):
            attn.prefill(torch.zeros(2, 3, 8), None, None, None, 0, **{name: 1})
    for bad in (torch.zeros(2, dtype=torch.int64), torch.zeros(3, dtype=torch.int32), torch.zeros(2, 1, dtype=torch.int32)):
        with pytest.raises(RuntimeError, match="q_lens must be int32"):
            attn.prefill(torch.zeros(2, 3, 8), None, None, None, 0, q_lens=bad)


def test_arguments_with_derivatives(fd):
    """Reverse mode while autograd records, forward mode always; queries, caches and fp8 scales alike."""
    from torch.autograd import forward_ad
    mk = lambda *s, dt=torch.bfloat16: torch.zeros(*s, dtype=dt)  # noqa: E731
    i32 = lambda *s: mk(*s, dt=torch.int32)  # noqa: E731

    def pre(q=mk(4, 8, 128), k=mk(6, 16, 2, 128), v=mk(6, 16, 2, 128), **kw):
        return fd.gqa_fwd_batch_prefill(q, k, v, i32(3), i32(2), i32(2, 4), 0.1, **kw)

    def shared(q=mk(4, 8, 128), k=mk(6, 16, 2, 128), v=mk(6, 16, 2, 128), **kw):
        return fd.gqa_fwd_batch_decode_shared_prefix(q, k, v, None, None, i32(4), i32(4, 2), i32(1), i32(1, 2), 0.1, **kw)

    for call in (pre, shared):
        for name, shape, dt in (("q", (4, 8, 128), torch.bfloat16), ("k", (6, 16, 2, 128), torch.bfloat16),
                                ("v", (6, 16, 2, 128), torch.bfloat16), ("k_scale", (2,), torch.float32),
                                ("v_scale", (2,), torch.float32)):
            other = {n: mk(2, dt=torch.float32) for n in ("k_scale", "v_scale")} if "scale" in name else {}
            leaf = mk(*shape, dt=dt).requires_grad_()
            with pytest.raises(RuntimeError, match="no backward"):
                call(**{**other, name: leaf})
            with torch.no_grad(), pytest.raises(RuntimeError, match="no CPU path"):      # allowed: the next check answers
                call(**{**other, name: leaf})
            with forward_ad.dual_level(), torch.no_grad():
                dual = forward_ad.make_dual(mk(*shape, dt=dt), mk(*shape, dt=dt))
                with pytest.raises(RuntimeError, match="forward-mode"):
                    call(**{**other, name: dual})
                with pytest.raises(RuntimeError, match="no CPU path"):
                    call(**other)


def test_the_most_forks_of_a_call(fd):
    import ctypes
    L, lib = fd._lib, fd.load_library()
    p, t = L.FdPagePool(), L.FdPageTables()
    p.k_cache = p.v_cache = t.block_table = t.kv_lens = t.page_refs = 0x10000
    p.k_page_bytes = p.v_page_bytes = p.k_page_stride = p.v_page_stride = 4096
    p.layers, p.num_pages, p.page_size, t.stride_table_bs, t.max_pages_per_seq, t.batch = 1, 8, 16, 4, 4, 40000
    n = 16385
    assert lib.fd_pages_fork(None, ctypes.byref(p), ctypes.byref(t), 0x10000, 0x10000, n, 0x10000, 0x10000, 12 * n) == -5
    assert b"16384" in lib.fd_last_error()


def test_hints_and_splits_count_by_value(fd, monkeypatch):
    """Given as tensors they may change in place between calls."""
    import importlib
    pre = importlib.import_module(fd.__name__ + ".kernels.prefill")
    seen = []
    monkeypatch.setattr(pre, "_prefill_image", lambda *a: (None, seen.append(a[-2:])))
    monkeypatch.setattr(pre, "_shared_image", lambda *a: (None, seen.append(a[-1])))
    mk = lambda *s, dt=torch.bfloat16: torch.zeros(*s, dtype=dt)  # noqa: E731
    i32 = lambda *s: mk(*s, dt=torch.int32)  # noqa: E731
    q, kv, a, b = mk(3, 8, 128), mk(6, 16, 2, 128), torch.tensor(5), torch.tensor(2)
    for x, y in ((5, 2), (2000, 2), (2000, 3)):
        a.fill_(x), b.fill_(y)
        for _ in range(2):
            fd.gqa_fwd_batch_prefill(q, kv, kv, i32(3), i32(2), i32(2, 4), 0.1, max_kv_len=a, kv_split=b)
            fd.gqa_fwd_batch_decode_shared_prefix(q, kv, kv, None, None, i32(3), i32(3, 2), i32(1), i32(1, 2), 0.1,
                                                  max_kv_len=a, max_prefix_len=b)
    assert seen == [(5, 2), (1024, 1024), (2000, 2), (2048, 1024), (2000, 3)]
    assert all(type(n) is int for pair in seen for n in pair)


def test_table_rows_that_overlap_are_refused(fd):
    """A page operator writes the table: an expanded row, or windows of one, would be several rows at once."""
    import ctypes
    L, lib = fd._lib, fd.load_library()
    t = L.FdPageTables()
    t.block_table = t.kv_lens = t.page_refs = 0x10000
    t.max_pages_per_seq, t.batch = 4, 3
    for stride in (0, 3):
        t.stride_table_bs = stride
        assert lib.fd_pages_reserve(None, ctypes.byref(t), 8, 16, None, 1, 0x10000) == -1 and b"apart" in lib.fd_last_error()
        assert lib.fd_pages_free(None, ctypes.byref(t), 8, 0x10000, 1) == -1 and b"apart" in lib.fd_last_error()
    t.batch = 1                                                  # one row: its stride means nothing
    assert lib.fd_pages_free(None, ctypes.byref(t), 8, None, 0) == 0
