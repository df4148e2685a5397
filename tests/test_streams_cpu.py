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


def weight(b, n=32, k=256):
    return b.Nvfp4Weight(torch.zeros((n, k // 2), dtype=torch.uint8), torch.zeros((n, k // 16), dtype=torch.uint8), torch.ones(1), device='cpu')


def layer(b):
    e = [(weight(b), weight(b), weight(b)) for _ in range(2)]
    L = b.MoeLayer(torch.zeros((2, 256), dtype=torch.bfloat16), torch.zeros(2), e, None, 1, 256, 32)
    L._ws[3] = torch.zeros(64, dtype=torch.uint8)                                    # kept from an earlier call
    return L


f32, b16 = lambda: torch.zeros(3, 256), lambda: torch.zeros((3, 256), dtype=torch.bfloat16)
CALLS = {
    'gemm': lambda b, s: b.gemm(weight(b), f32(), stream=s),
    'gemm with scratch': lambda b, s: b.gemm(weight(b), f32(), stream=s, ws=b.split_workspace(3, 256, 'cpu', s)),
    'gemm of a plain matrix': lambda b, s: b.gemm(b16(), f32(), stream=s),
    'gemm_bf16': lambda b, s: b.gemm_bf16(weight(b), b16(), stream=s),
    'gemm_bf16_exact': lambda b, s: b.gemm_bf16_exact(weight(b), b16(), stream=s),
    'quantize_tokens': lambda b, s: b.quantize_tokens(f32(), stream=s),
    'dense_mlp': lambda b, s: b.dense_mlp(f32(), weight(b), weight(b), weight(b), stream=s),
    'gemv_multi': lambda b, s: b.gemv_multi([weight(b), weight(b)], f32(), 3, stream=s),
    'f32_to_bf16': lambda b, s: b.f32_to_bf16(f32(), stream=s),
    'bf16_to_f32': lambda b, s: b.bf16_to_f32(b16(), stream=s),
    'quantize': lambda b, s: b.quantize(b16(), stream=s),
    'dequantize': lambda b, s: b.dequantize(weight(b), stream=s),
    'moe_route': lambda b, s: b.moe_route(layer(b), f32(), stream=s),
    'moe_forward': lambda b, s: b.moe_forward(layer(b), f32(), stream=s),
    'moe_experts': lambda b, s: b.moe_experts(layer(b), f32(), torch.zeros(3, 1, dtype=torch.int32), torch.zeros(3, 1), stream=s),
    'moe_forward_static': lambda b, s: b.moe_forward_static(layer(b), f32(), stream=s),
    'EpContext.forward': lambda b, s: b.EpContext(layer(b), layer(b), None, 0, 1, 3).forward(f32(), stream=s),
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


def test_codes_of_tokens_are_put_in_order_behind_their_kernel(calls, monkeypatch):
    """quantize_tokens rearranges what its kernel wrote: on the kernel's stream."""
    b, made, recorded = calls
    on, copy = [], torch.Tensor.copy_
    monkeypatch.setattr(torch.Tensor, 'copy_', lambda t, *a: (on.append(torch.cuda.current_stream()), copy(t, *a))[1])
    contiguous = torch.Tensor.contiguous
    monkeypatch.setattr(torch.Tensor, 'contiguous', lambda t, *a: (on.append(torch.cuda.current_stream()), contiguous(t, *a))[1])
    other = Stream()
    b.quantize_tokens(torch.zeros(3, 512), stream=other)
    assert on and all(s is other for s in on)
