"""CPU-only: where the wrappers of prompt attention and of the page operators take memory for work on a given stream."""
import contextlib
import importlib

import pytest
import torch


class _Stream:
    device = torch.device("cuda", 0)
    cuda_stream = 0


def test_memory_for_a_stream_comes_from_its_pool(fd, monkeypatch):
    pre = importlib.import_module(fd.__name__ + ".kernels.prefill")
    inside, recorded, allocated = [], [], []

    @contextlib.contextmanager
    def enter(s):
        inside.append(s)
        try:
            yield
        finally:
            inside.pop()

    class Tensor(torch.Tensor):
        def record_stream(self, s):
            recorded.append(s)

    def empty(*shape, device=None, **kw):
        allocated.append(inside[-1] if inside else "current")
        return torch.zeros(*shape, **kw).as_subclass(Tensor)

    monkeypatch.setattr(torch.cuda, "stream", enter)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: "current")
    monkeypatch.setattr(torch, "empty", empty)
    side = _Stream()
    pre._new(5, torch.int32, side.device, None)
    assert allocated == ["current"] and not recorded
    pre._new(5, torch.int32, side.device, side)                          # a workspace: freed into the pool of its stream
    pre._new(5, torch.int32, side.device, side, returned=True)           # a result: the caller uses it on the current stream
    pre._workspace(None, 64, side.device, side)
    assert allocated == ["current"] + [side] * 3 and recorded == ["current"]


def test_a_stream_of_another_device_is_refused(fd):
    pre = importlib.import_module(fd.__name__ + ".kernels.prefill")
    with pytest.raises(RuntimeError, match="another device"):
        pre._launch(lambda *a: 0, torch.device("cuda", 1), _Stream())


def test_the_block_enters_the_stream_before_any_of_its_work(fd, monkeypatch):
    """``prefill`` and ``fwd``: the first projection already runs on the given stream."""
    inside = []

    @contextlib.contextmanager
    def enter(s):
        inside.append(s)
        try:
            yield
        finally:
            inside.pop()

    class Reached(Exception):
        pass

    def linear(*args):
        seen.append(inside[-1] if inside else "current")
        raise Reached

    monkeypatch.setattr(torch.cuda, "stream", enter)
    monkeypatch.setattr(torch.nn.functional, "linear", linear)
    attn, side, seen = fd.layers.TP_Attn(), _Stream(), []
    for method, n in ((attn.prefill, 3), (attn.fwd, 1)):
        for kw in ({"stream": side}, {}):
            with pytest.raises(Reached):
                method(torch.zeros(2, n, 8), None, None, None, 0, **kw)
    assert seen == [side, "current"] * 2
