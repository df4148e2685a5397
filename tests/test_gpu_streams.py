"""Calls on another stream that allocate their own outputs and scratch, while the current stream still writes memory that was freed."""
import numpy as np
import pytest
import torch

from util import pkg
from test_gpu_moe import build_layer

pytestmark = pytest.mark.gpu


def weight(P, n, k, seed):
    g = torch.Generator(device='cuda').manual_seed(seed)
    return P.quantize((torch.randn((n, k), generator=g, device='cuda') * 0.02).to(torch.bfloat16))


def paths(P):
    """name -> call(stream) -> outputs"""
    g = torch.Generator(device='cuda').manual_seed(1)
    x = torch.randn((40, 1024), generator=g, device='cuda')
    xb = x.to(torch.bfloat16)
    gate, up, down = weight(P, 512, 1024, 1), weight(P, 512, 1024, 2), weight(P, 1024, 512, 3)
    out = lambda r: [r] if torch.is_tensor(r) else list(r)
    return {
        'gemm': lambda s: out(P.gemm(gate, x[:8], stream=s)),
        'gemm_bf16': lambda s: out(P.gemm_bf16(gate, xb, stream=s)),
        'gemm_bf16_exact': lambda s: out(P.gemm_bf16_exact(gate, xb, stream=s)),
        'dense_mlp': lambda s: out(P.dense_mlp(x, gate, up, down, stream=s)),
        'gemv_multi': lambda s: out(P.gemv_multi([gate, up], x[:4], 4, stream=s)),
        'quantize_tokens': lambda s: out(P.quantize_tokens(x, stream=s)),
        'f32_to_bf16': lambda s: out(P.f32_to_bf16(x, stream=s)),
        'quantize': lambda s: [P.quantize(xb, stream=s).packed],
        'dequantize': lambda s: out(P.dequantize(gate, stream=s)),
    }


NAMES = ['gemm', 'gemm_bf16', 'gemm_bf16_exact', 'dense_mlp', 'gemv_multi', 'quantize_tokens', 'f32_to_bf16', 'quantize', 'dequantize']


def occupy(sizes):
    """The current stream sleeps and then writes tensors of these sizes, which are free when this returns."""
    old = [torch.zeros(n, dtype=torch.uint8, device='cuda') for n in sizes for _ in range(4)]
    torch.cuda.synchronize()
    torch.cuda._sleep(20_000_000)
    for o in old:
        o.fill_(255)


@pytest.mark.parametrize('name', NAMES)
def test_a_call_on_another_stream_gets_none_of_the_current_one_s_memory(name):
    P = pkg()
    call, s = paths(P)[name], torch.cuda.Stream()
    want = [o.clone() for o in call(None)]
    torch.cuda.synchronize()
    sizes = [o.nbytes for o in want] + [P.gemm_bf16_workspace(40, 1024, 'cuda').nbytes, P.dense_mlp_workspace(40, 1024, 512, 'cuda').nbytes]
    occupy(sizes)
    got = call(s)
    torch.cuda.synchronize()
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(got, want))


@pytest.mark.parametrize('M', [1, 5, 20])
def test_a_layer_s_first_call_is_on_another_stream(M):
    """The scratch that a layer keeps comes from the current stream's memory, whose last user may still be at work."""
    P = pkg()
    layer, _ = build_layer(1024, 512, 16, 4, seed=3)
    x = torch.from_numpy(np.random.default_rng(M).normal(0, 1, (M, 1024)).astype(np.float32)).cuda()
    want = [o.clone() for o in P.moe_forward(layer, x)]
    n = layer.workspace(M).nbytes
    layer._ws.clear()
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    occupy([n] + [o.nbytes for o in want])
    got = P.moe_forward(layer, x, stream=s)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert P.device_status() == 0


def test_calls_on_a_side_stream_of_a_captured_graph():
    """A captured graph forks, calls on the side stream with outputs and scratch of their own, and joins; replayed on new inputs."""
    P = pkg()
    g = torch.Generator(device='cuda').manual_seed(5)
    w = (torch.randn((700, 1024), generator=g, device='cuda') * 0.02).to(torch.bfloat16)
    W, Wn = P.i8_quantize(w), weight(P, 512, 1024, 5)
    x = torch.randn((40, 1024), generator=g, device='cuda')
    t = torch.zeros((40, 1), dtype=torch.int32, device='cuda')

    def calls(s):
        y = P.i8_gemm(W, x, stream=s)
        return [y, P.i8_gemm(W, P.i8_quantize(x, stream=s), stream=s), *P.token_logprobs(y, t, 4, stream=s), P.gemm(Wn, x[:8], stream=s)]

    calls(None)
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph):
        side.wait_stream(torch.cuda.current_stream())
        got = calls(side)
        torch.cuda.current_stream().wait_stream(side)
    for seed in (6, 7):
        x.copy_(torch.randn((40, 1024), generator=g.manual_seed(seed), device='cuda'))
        graph.replay()
        other = [torch.full((1 << 16,), 7.0, device='cuda') for _ in range(4)]            # memory that is not the graph's
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, calls(None)))
        del other
