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
