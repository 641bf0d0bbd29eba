"""Where a step is captured: on a stream of the GPU that its tensors are on, whichever is the current one.  torch's
own stream for captures is on the GPU that was current when it was first asked for; a step on another GPU would leave a graph
of nothing.  On the CPU, with stand-ins that note which streams are used."""
import contextlib

import pytest
import torch


class _Stream:
    def __init__(self, device=None):
        self.device = device

    def wait_stream(self, other):
        pass


@pytest.fixture
def used(monkeypatch):
    now, seen = [None], []

    @contextlib.contextmanager
    def on(stream):
        now.append(stream)
        yield
        now.pop()

    @contextlib.contextmanager
    def graph(g, pool=None, stream=None, **kw):
        with on(stream):
            yield

    monkeypatch.setattr(torch.cuda, "Stream", _Stream)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: _Stream(device))
    monkeypatch.setattr(torch.cuda, "stream", on)
    monkeypatch.setattr(torch.cuda, "CUDAGraph", lambda: None)
    monkeypatch.setattr(torch.cuda, "graph", graph)
    return now, seen


def test_steps_with_state_are_captured_on_their_gpu(used):
    from fxlm.model import _captured
    now, seen = used
    state = torch.zeros(3)
    _captured(lambda: seen.append(now[-1]), [state])
    assert len(seen) == 3 and all(s is not None and s.device == state.device for s in seen)


def test_decode_steps_are_captured_on_their_gpu(used):
    from fxlm.model import _DecodeGraph
    now, seen = used

    class Model:
        pos_emb = torch.zeros(8, 4)

        def _decode(self, tok, cache, pos, lens):
            seen.append(now[-1])

    k = torch.zeros(2, 8, 1, 4)
    _DecodeGraph(Model(), [(k, k.clone())], 2)
    assert len(seen) == 3 and all(s is not None and s.device == k.device for s in seen)
