"""A dense cache's own block table: captured without a call before, read on another stream than the one that made it."""
import pytest
import torch

from test_gpu_serving import BF16, DEV, make_block, positions

pytestmark = pytest.mark.gpu


def test_capture_first_then_eager_then_replay(fd):
    """The graph's first table is filled by its replays only: an eager call in between has a table of its own."""
    gen = torch.Generator().manual_seed(7)
    B, hidden, Hq, Hkv, D = 11, 128, 4, 2, 64        # (a batch that no other test has)
    attn, tab = make_block(fd, hidden, Hq, Hkv, D, gen)
    kw = dict(num_layers=1, batch_size=B, max_length=64, kv_heads=Hkv, head_dim=D, dtype=BF16, world_size=1)
    x = torch.randn(B, 5, hidden, generator=gen).to(BF16).to(DEV)
    caches = [fd.layers.KV_Cache(**kw) for _ in range(3)]
    pos = positions(caches[0], 5, B)
    paged = fd.layers.PagedKV_Cache(page_size=16, **kw)
    torch.nn.functional.linear(x, attn.wqkv)         # (the library's own workspace, before the capture)
    want = attn.prefill(x, pos, tab, paged, 0)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = attn.prefill(x, pos, tab, caches[0], 0)
    assert torch.equal(attn.prefill(x, pos, tab, caches[1], 0), want)
    for _ in range(3):
        with torch.inference_mode():
            y.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want) and torch.equal(caches[0].k_cache, caches[1].k_cache)
        assert torch.equal(attn.prefill(x, pos, tab, caches[2], 0), want)


def test_every_stream_fills_the_table_it_reads(fd):
    from importlib import import_module
    app = import_module(fd.__name__ + ".kernels.kv_append")
    a, side = app._dense_block_table(torch.device("cuda", 0), 13), torch.cuda.Stream()
    with torch.cuda.stream(side):
        b = app._dense_block_table(torch.device("cuda", 0), 13)
        assert app._dense_block_table(torch.device("cuda", 0), 13) is b
    assert a is not b and app._dense_block_table(torch.device("cuda", 0), 13) is a
    torch.cuda.synchronize()
    assert a[:, 0].tolist() == b[:, 0].tolist() == list(range(13))
