"""CPU-only: calls with ``stream=`` switch to the stream for all they do, memory included, and back."""
import importlib

import pytest
import torch


class _Stream:
    def __init__(self, handle, index=0):
        self.cuda_stream, self.device, self.device_index = handle, torch.device("cuda", index), index


@pytest.fixture
def streams(fd, monkeypatch):
    """The current stream as the wrappers see it; `now[0]`."""
    flash = importlib.import_module(fd.__name__ + ".kernels.flash_decode")
    now = [_Stream(1)]
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: now[0])
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "set_stream", lambda s: now.__setitem__(0, s))
    monkeypatch.setattr(flash, "stream_handle", lambda stream=None, index=None: (stream or now[0]).cuda_stream)
    return flash, now


def test_a_call_runs_on_its_stream_and_comes_back(streams):
    flash, now = streams
    first, side, seen = now[0], _Stream(2), []

    class Result(torch.Tensor):
        def record_stream(self, s):
            seen.append(("used on", s))

    def work(*args, **kw):
        seen.append(now[0])
        return (torch.zeros(1).as_subclass(Result), None) if kw else None

    flash._on(None, work)
    flash._on(first, work, 1, a=2)                               # the current one: nothing to do
    assert seen == [first, first] and now[0] is first
    del seen[:]
    flash._on(side, work, torch.zeros(2), a=2)                   # what comes back may be used on the current one
    assert seen == [side, ("used on", first)] and now[0] is first
    with pytest.raises(ZeroDivisionError):
        flash._on(side, lambda: 1 // 0)
    assert now[0] is first


class _OnGpu(torch.Tensor):
    is_cuda = True
    device = torch.device("cuda", 1)


def test_a_stream_of_another_device_is_refused(streams):
    flash, now = streams
    with pytest.raises(RuntimeError, match="a stream of cuda:0"):
        flash._on(_Stream(2), lambda *a: None, None, torch.zeros(2).as_subclass(_OnGpu))


def test_every_entry_point_is_on_its_stream_before_it_does_anything(fd, streams, monkeypatch):
    flash, now = streams
    pre, pages, app = (importlib.import_module(f"{fd.__name__}.kernels.{m}") for m in ("prefill", "pages", "kv_append"))
    first, side, seen = now[0], _Stream(2), []

    class Reached(Exception):
        pass

    def reached(*args, **kw):
        seen.append(now[0])
        raise Reached

    for module, name in ((pre, "_check_no_grad"), (pages, "_checked"), (flash, "load_library"), (app, "load_library"),
                         (flash, "_require_cuda"), (torch.nn.functional, "linear")):
        monkeypatch.setattr(module, name, reached)
    q, i = torch.zeros(2, 1, 4, 64), torch.zeros(2, dtype=torch.int32)
    attn = fd.layers.TP_Attn()
    calls = [lambda **kw: fd.gqa_fwd_batch_prefill(q, q, q, i, None, None, 0.1, **kw),
             lambda **kw: fd.gqa_fwd_batch_decode_shared_prefix(q, q, q, None, None, i, i, i, i, 0.1, **kw),
             lambda **kw: fd.paged_kv_copy(q, q, i, i, **kw), lambda **kw: fd.paged_kv_reserve(i[None], i, i, 1, 16, **kw),
             lambda **kw: fd.paged_kv_fork(q, q, i, i, i, i, i, **kw), lambda **kw: fd.paged_kv_free(i, i, i, i, **kw),
             lambda **kw: fd.paged_kv_compact(q, q, i, i, **kw),
             lambda **kw: fd.gqa_fwd_batch_decode(q[:, 0], q, q, None, None, i, i[None], 0.1, **kw),
             lambda **kw: fd.gqa_fwd_batch_decode_intra_rank(q[:, 0], q, q, None, None, i, i[None], 0.1, **kw),
             lambda **kw: fd.rope_kv_append(q, q, q, q, i, i, **kw),
             lambda **kw: fd.flash_attn_with_kvcache(q, q, q, k=q, v=q, cache_seqlens=i, auto_order=False, **kw),
             lambda **kw: attn.prefill(torch.zeros(2, 3, 8), None, None, None, 0, **kw),
             lambda **kw: attn.fwd(torch.zeros(2, 1, 8), None, None, None, 0, **kw)]
    monkeypatch.setattr(app, "_dense_block_table", lambda device, n: i[:, None])
    for k, call in enumerate(calls):
        for kw in ({"stream": side}, {}, {"stream": None}):
            with pytest.raises(Reached):
                call(**kw)
            assert now[0] is first and seen.pop() is (side if kw.get("stream") else first), (k, kw)
