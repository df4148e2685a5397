"""Whose memory a call on another stream allocates: every output and scratch of its own has to be that stream's, and recorded for the
current stream, which the caller goes on with."""
import contextlib
import importlib

import pytest
import torch

import __graft_entry__ as G
from util import pkg

HERE = object()


class FakeLib:
    """Every entry point succeeds; sizes are small."""
    def __getattr__(self, name):
        return (lambda *a: 1 << 16) if name.endswith('_bytes') else (lambda *a: 0)


@pytest.fixture
def calls(monkeypatch):
    """(the binding, [(tensor, stream it was allocated on)], {address of a recorded tensor: streams})"""
    pkg()
    b = importlib.import_module(G.PKG_NAME + '.binding')
    now, made, recorded, empty = [HERE], [], {}, torch.empty

    @contextlib.contextmanager
    def on(stream):
        now.append(now[-1] if stream is None else stream)
        yield
        now.pop()

    def spy(*a, **k):
        k.pop('device', None)
        t = empty(*a, **k)
        made.append((t, now[-1]))
        return t

    monkeypatch.setattr(torch, 'empty', spy)
    monkeypatch.setattr(torch.cuda, 'stream', on)
    monkeypatch.setattr(torch.cuda, 'current_stream', lambda *a: now[-1])
    monkeypatch.setattr(torch.Tensor, 'record_stream', lambda t, s: recorded.setdefault(id(t), []).append(s), raising=False)
    monkeypatch.setattr(torch._C, '_cuda_getDevice', lambda: -1, raising=False)      # where CPU tensors say they are
    monkeypatch.setattr(torch._C, '_cuda_getCurrentRawStream', lambda d: 0, raising=False)
    monkeypatch.setattr(b, '_stream', lambda s: 0)
    monkeypatch.setattr(b, '_device', lambda *t: None)
    monkeypatch.setattr(b, 'lib', FakeLib)
    return b, made, recorded


class Stream:
    cuda_stream = 0


def rows(b, n, k):
    return b.I8Rows(torch.zeros((n, (k + 31) // 32 * 32), dtype=torch.int8), torch.zeros(n), k)


CALLS = {
    'i8_quantize': lambda b, s: b.i8_quantize(torch.zeros(3, 40), stream=s),
    'i8_gemm': lambda b, s: b.i8_gemm(rows(b, 5, 40), torch.zeros(3, 40), stream=s),
    'i8_gemm with scratch': lambda b, s: b.i8_gemm(rows(b, 5, 40), torch.zeros(3, 40), ws=torch.zeros(4096, dtype=torch.uint8), stream=s),
    'i8_gemm on rows': lambda b, s: b.i8_gemm(rows(b, 5, 40), rows(b, 3, 40), dtype=torch.bfloat16, stream=s),
    'token_logprobs': lambda b, s: b.token_logprobs(torch.zeros(3, 40), torch.zeros((3, 2), dtype=torch.int32), 4, stream=s),
}


def hold(calls, call):
    b, made, recorded = calls
    made.clear()
    call(b, None)
    assert made and all(s is HERE for _, s in made) and not recorded
    made.clear()
    other = Stream()
    call(b, other)
    assert made and all(s is other for _, s in made)
    assert all(recorded.get(id(t)) == [HERE] for t, _ in made)


@pytest.mark.parametrize('name', CALLS)
def test_what_a_call_on_another_stream_allocates(calls, name):
    hold(calls, CALLS[name])
