"""Rows of 8-bit integers and their products on the GPU.

The rule of the codes and the epilogue are single f32 operations and the sum is a whole number below 2^31, so every output has
exactly one right value: the oracle does the same steps in numpy (sums in 64 bits) and outputs are compared bit for bit."""
import numpy as np
import pytest
import torch

from util import pkg
from test_gpu_early_start import late_copy

pytestmark = pytest.mark.gpu


def gen(seed):
    return torch.Generator().manual_seed(seed)


def rows_of(x):
    """(codes int8 [rows, K], scale f32 [rows]) of a CPU tensor, by the rule."""
    x = x.float().numpy()
    bad = ~np.isfinite(x).all(1)
    a = np.maximum(np.abs(np.where(bad[:, None], 0, x)).max(1), np.float32(2.0 ** -119)).astype(np.float32)
    inv, scale = np.float32(127) / a, a / np.float32(127)
    q = np.rint(np.where(bad[:, None], 0, x) * inv[:, None])
    assert np.abs(q).max() <= 127
    return q.astype(np.int8), np.where(bad, np.float32(np.nan), scale).astype(np.float32)


def product(qx, sx, qw, sw, dtype):
    acc = qx.astype(np.float64) @ qw.astype(np.float64).T                    # whole numbers below 2^53
    y = (acc.astype(np.float32) * sx[:, None]) * sw[None, :]
    return torch.from_numpy(y).to(dtype)


def same(a, b):
    """Equal bit for bit; NaN equals NaN."""
    assert a.shape == b.shape and a.dtype == b.dtype
    bits = torch.int16 if a.dtype == torch.bfloat16 else torch.int32 if a.dtype == torch.float32 else a.dtype
    a, b = a.cpu(), b.cpu()
    nan = a.isnan() & b.isnan()
    return bool(((a.view(bits) == b.view(bits)) | nan).all())


def inputs(M, N, K, seed, dtype=torch.float32):
    g = gen(seed)
    x = torch.randn((M, K), generator=g) * torch.exp(torch.randn((M, 1), generator=g))
    w = torch.randn((N, K), generator=g) * 0.02 * torch.exp(0.3 * torch.randn((N, 1), generator=g))
    return x.to(dtype), w.to(torch.bfloat16)


# ---- the rows ------------------------------------------------------------------------------------

@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('M,K', [(1, 1), (3, 7), (2, 16), (5, 17), (4, 4096), (3, 8191), (2, 8192), (2, 8200), (2, 30001), (1, 65536), (700, 96)])
def test_rows_are_the_rule_s(M, K, dtype):
    P = pkg()
    x, _ = inputs(M, 1, K, M + K, dtype)
    q, s = rows_of(x)
    r = P.i8_quantize(x.cuda())
    assert r.q.shape == (M, (K + 31) // 32 * 32)
    assert np.array_equal(r.q[:, :K].cpu().numpy(), q) and np.array_equal(r.scale.cpu().numpy(), s)
    assert not r.q[:, K:].any()


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_rows_at_the_edges_of_the_type(dtype):
    """Zeros, the smallest and largest numbers, halves between two codes, signed zeros, infinities and NaN."""
    P = pkg()
    K = 40
    x = torch.zeros((12, K))
    x[1, 3] = 2.0 ** -126
    x[2, :] = torch.linspace(-1, 1, K) * 2.0 ** -120
    x[3, :] = torch.linspace(-1, 1, K) * 3.3e38
    x[4, :] = torch.arange(K) - 20.5
    x[4, 0] = 127.0                                                     # a = 127: codes are the numbers, halves go to even
    x[5, 7], x[5, 8] = -0.0, 1.0
    x[6, 11] = float('inf')
    x[7, 39] = float('nan')
    x[8, 0] = float('-inf')
    x[9, :] = 1.0
    x[10, :] = -1.0
    x[11, 5] = 2.0 ** -119
    x = x.to(dtype)
    q, s = rows_of(x)
    r = P.i8_quantize(x.cuda())
    assert np.array_equal(r.q[:, :K].cpu().numpy(), q)
    assert np.array_equal(r.scale.cpu().numpy(), s, equal_nan=True)
    assert r.scale[6:9].isnan().all() and torch.isfinite(r.scale[[0, 1, 2, 3, 4, 5, 9, 10, 11]]).all()


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('off,ld', [(0, 104), (0, 101), (1, 104), (3, 99), (8, 128)])
def test_rows_of_strided_and_unaligned_tensors(dtype, off, ld):
    P = pkg()
    M, K = 6, 90
    big = torch.randn(M * ld + off + 8, generator=gen(off + ld)).to(dtype).cuda()
    x = torch.as_strided(big, (M, K), (ld, 1), off)
    q, s = rows_of(x.cpu())
    r = P.i8_quantize(x)
    assert np.array_equal(r.q[:, :K].cpu().numpy(), q) and np.array_equal(r.scale.cpu().numpy(), s)


def test_rows_behind_the_last_stay():
    P = pkg()
    x = torch.randn((5, 33), generator=gen(3)).cuda()
    q, s = torch.full((7, 64), 77, dtype=torch.int8, device='cuda'), torch.full((7,), 7.0, device='cuda')
    out = P.I8Rows(q[:5], s[:5], 33)
    P.i8_quantize(x, out=out)
    assert (q[5:] == 77).all() and (s[5:] == 7).all()


# ---- the product ---------------------------------------------------------------------------------

SHAPES = [(1, 1, 1), (1, 128, 4096), (1, 4096, 256), (2, 7, 17), (3, 130, 31), (4, 1000, 2048), (5, 129, 127), (7, 64, 12288), (8, 300, 640), (9, 255, 130),
          (12, 5003, 64), (15, 33, 1040), (16, 257, 128), (17, 512, 384), (31, 200, 2051), (33, 129, 100), (64, 640, 512), (65, 127, 2048), (100, 300, 2051),
          (128, 128, 128), (129, 1000, 272), (200, 4096, 160), (255, 130, 900), (257, 385, 1025), (300, 2000, 513), (513, 700, 256), (777, 1003, 320),
          (1030, 513, 208)]


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('off', range(1, 8))
def test_rows_at_every_place(off, dtype):
    """Every distance from a 16-byte boundary, lengths around the vectors that hold a row's ends; NaN around the rows."""
    P = pkg()
    for K in (1, 5, 8, 9, 15, 16, 17, 23, 24, 25, 31, 33, 63, 100, 1027, 4090, 4103, 8195, 9001):
        x, _ = inputs(5, 1, K, 7 * K + off, dtype)
        for ld in (K, K + 1, K + 3):
            flat = torch.full((off + 5 * ld + 9,), float('nan'), dtype=dtype, device='cuda')
            view = flat[off:off + 5 * ld].view(5, ld)[:, :K]
            view.copy_(x)
            r, (q, s) = P.i8_quantize(view), rows_of(x)
            assert np.array_equal(r.q[:, :K].cpu().numpy(), q) and np.array_equal(r.scale.cpu().numpy(), s) and not r.q[:, K:].any()


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('M,K,ld', [(601, 1, 1), (297, 64, 64), (330, 100, 104), (1201, 33, 33), (1187, 511, 513), (1190, 1023, 1025), (1500, 512, 515),
                                    (299, 1024, 1024), (1203, 2047, 2049), (301, 2048, 2048)])
def test_many_short_rows(M, K, ld, dtype):
    P = pkg()
    x, _ = inputs(M, 1, K, M + K, dtype)
    x[3], x[M - 1, K // 2], x[M - 2, 0], x[M - 3, K - 1] = 0, float('inf'), float('nan'), 1e30
    big = torch.zeros((M, ld), dtype=dtype, device='cuda')
    big[:, :K] = x.cuda()
    pitch = (K + 31) // 32 * 32
    q, s = torch.full((M + 4, pitch), 77, dtype=torch.int8, device='cuda'), torch.full((M + 4,), 7.0, device='cuda')
    P.i8_quantize(big[:, :K], out=P.I8Rows(q[:M], s[:M], K))
    wq, ws = rows_of(x)
    assert np.array_equal(q[:M, :K].cpu().numpy(), wq) and np.array_equal(s[:M].cpu().numpy(), ws, equal_nan=True)
    assert not q[:M, K:].any() and (q[M:] == 77).all() and (s[M:] == 7).all()


@pytest.mark.parametrize('M,N,K', SHAPES)
def test_product_is_exact(M, N, K):
    P = pkg()
    i = SHAPES.index((M, N, K))
    x, w = inputs(M, N, K, i, (torch.float32, torch.bfloat16)[i & 1])
    qx, sx = rows_of(x)
    qw, sw = rows_of(w)
    W = P.i8_quantize(w.cuda())
    for dtype in (torch.float32, torch.bfloat16):
        want = product(qx, sx, qw, sw, dtype)
        assert same(P.i8_gemm(W, x.cuda(), dtype=dtype), want)
        assert same(P.i8_gemm(W, P.i8_quantize(x.cuda()), dtype=dtype), want)
    assert P.device_status() == 0


# On 148 multiprocessors these go to pairs of CTAs, in tiles of 64, 96, 128, 160, 160, 192, 192, 224, 224, 256 and 256 tokens; one, two or three
# items a pair (up to 20, 28, 114, 50, 200, 50, 190, 50, 180, 50 and 180 items for 74 pairs).
PAIRS = [(289, 1010, 1029), (644, 1001, 1029), (338, 9523, 1300), (290, 6310, 1029), (580, 12576, 1029), (323, 6356, 1029), (808, 9505, 1029),
         (417, 6342, 771), (840, 11268, 771), (453, 6359, 771), (897, 11280, 771)]


@pytest.mark.parametrize('M,N,K', PAIRS)
def test_product_on_pairs_is_exact(M, N, K):
    P = pkg()
    i = PAIRS.index((M, N, K))
    x, w = inputs(M, N, K, 100 + i, (torch.float32, torch.bfloat16)[i & 1])
    want = product(*rows_of(x), *rows_of(w), torch.float32)
    W, X = P.i8_quantize(w.cuda()), P.i8_quantize(x.cuda())
    for dtype in (torch.float32, torch.bfloat16):
        buf = torch.full((M * N + 999,), 3.0, dtype=dtype, device='cuda')
        P.i8_gemm(W, x.cuda(), buf[:M * N].view(M, N))
        assert same(buf[:M * N].view(M, N), want.to(dtype)) and (buf[M * N:] == 3).all()
        assert same(P.i8_gemm(W, X, dtype=dtype), want.to(dtype))
    assert P.device_status() == 0


# Up to 8 rows: a warp's slice of K in several turns of loads (K above 4096, the last turn part full), and more units of weight rows to a CTA than
# its partial sums have room for at once (64 / M).
@pytest.mark.parametrize('M,N,K', [(1, 301, 4097), (1, 4100, 5003), (1, 77, 8192), (1, 300, 12288), (2, 200, 8200), (1, 130, 30000), (2, 97, 20001), (3, 500, 12289),
                                   (4, 64, 12288), (8, 160, 6200), (1, 160001, 192), (2, 154880, 256), (3, 50021, 100), (5, 60007, 300), (7, 43001, 129),
                                   (8, 40001, 520), (8, 20000, 4500),
                                   (2, 300, 12288), (1, 130, 18000), (1, 130, 24000), (4, 300, 6500), (3, 70, 8000), (8, 50, 4095)])
def test_few_rows_with_long_sums_and_many_outputs(M, N, K):
    P = pkg()
    x, w = inputs(M, N, K, M + N + K, (torch.float32, torch.bfloat16)[K & 1])
    want = product(*rows_of(x), *rows_of(w), torch.float32)
    W, X = P.i8_quantize(w.cuda()), P.i8_quantize(x.cuda())
    for dtype in (torch.float32, torch.bfloat16):
        assert same(P.i8_gemm(W, x.cuda(), dtype=dtype), want.to(dtype))
        assert same(P.i8_gemm(W, X, dtype=dtype), want.to(dtype))


def test_few_rows_with_weights_past_32_bits():
    """More than 2^31 bytes of weights in the kernel of few rows: one row quantised in the kernel, and finished rows."""
    P = pkg()
    N, K = 180001, 12288
    g = torch.Generator(device='cuda').manual_seed(2)
    q = torch.randint(-127, 128, (N, K), generator=g, device='cuda', dtype=torch.int8)
    sw = torch.rand(N, generator=g, device='cuda')
    W = P.I8Rows(q, sw, K)
    for M in (1, 2):
        x = torch.randn((M, K), generator=g, device='cuda')
        y = P.i8_gemm(W, x if M == 1 else P.i8_quantize(x)).cpu()
        for a in (0, N // 2, N - 200):
            assert same(y[:, a:a + 200].contiguous(), product(*rows_of(x.cpu()), q[a:a + 200].cpu().numpy(), sw[a:a + 200].cpu().numpy(), torch.float32))


@pytest.mark.parametrize('M', [1, 4, 20, 150, 520])
def test_largest_sums(M):
    """Codes of the caller's own, -128 among them, at the longest K: sums up to 2^30."""
    P = pkg()
    N, K = 140, 65536
    g = gen(M)
    qx = torch.randint(-128, 128, (M, K), generator=g, dtype=torch.int8)
    qw = torch.randint(-128, 128, (N, K), generator=g, dtype=torch.int8)
    qx[0], qw[0], qw[1] = -128, -128, 127
    sx, sw = torch.rand(M, generator=g), torch.rand(N, generator=g)
    y = P.i8_gemm(P.I8Rows(qw.cuda(), sw.cuda(), K), P.I8Rows(qx.cuda(), sx.cuda(), K))
    assert same(y, product(qx.numpy(), sx.numpy(), qw.numpy(), sw.numpy(), torch.float32))


@pytest.mark.parametrize('M', [1, 8, 30, 300])
def test_bytes_past_k_are_not_used(M):
    P = pkg()
    N, K = 200, 1029
    x, w = inputs(M, N, K, M)
    W, X = P.i8_quantize(w.cuda()), P.i8_quantize(x.cuda())
    want = P.i8_gemm(W, X)
    W.q[:, K:], X.q[:, K:] = 113, -77
    assert same(P.i8_gemm(W, X), want)


@pytest.mark.parametrize('M', [2, 9, 40, 300])
def test_rows_without_a_finite_scale_and_rows_of_zeros(M):
    P = pkg()
    x, w = inputs(M, 150, 700, M)
    x[0, 5], x[M - 1] = float('inf'), 0.0
    if M > 2:
        x[1, 699] = float('nan')
    w[3, 2] = float('nan')
    y = P.i8_gemm(P.i8_quantize(w.cuda()), x.cuda()).cpu()
    qx, sx = rows_of(x)
    qw, sw = rows_of(w)
    assert same(y, product(qx, sx, qw, sw, torch.float32))
    assert y[0].isnan().all() and y[:, 3].isnan().all() and (y[M - 1, torch.arange(150) != 3] == 0).all()


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_a_row_does_not_depend_on_its_batch(dtype):
    P = pkg()
    x, w = inputs(600, 1100, 1300, 5)
    W, xd = P.i8_quantize(w.cuda()), x.cuda()
    whole = P.i8_gemm(W, xd, dtype=dtype)
    for M in (1, 2, 5, 8, 9, 16, 17, 33, 70, 129, 300):
        assert same(P.i8_gemm(W, xd[:M], dtype=dtype), whole[:M])


@pytest.mark.parametrize('M', [1, 3, 8, 9, 40, 260])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_what_lies_behind_the_output_stays(M, dtype):
    P = pkg()
    x, w = inputs(M, 135, 300, M)
    buf = torch.full((M * 135 + 4096,), 3.0, dtype=dtype, device='cuda')
    y = buf[1:1 + M * 135].view(M, 135)                                 # at its type's alignment only
    P.i8_gemm(P.i8_quantize(w.cuda()), x.cuda(), y)
    assert same(y, product(*rows_of(x), *rows_of(w), dtype))
    assert buf[0] == 3 and (buf[1 + M * 135:] == 3).all()


@pytest.mark.parametrize('M', [1, 6, 33])
def test_strided_activations(M):
    P = pkg()
    x, w = inputs(M, 77, 333, M)
    big = torch.full((M, 401), 1e9)
    big[:, 5:338] = x
    assert same(P.i8_gemm(P.i8_quantize(w.cuda()), big.cuda()[:, 5:338]), product(*rows_of(x), *rows_of(w), torch.float32))


def test_offsets_past_32_bits():
    """A weight matrix and an output of more than 2^31 elements: the first and last rows are right."""
    P = pkg()
    N, K, M = 140001, 16384, 3
    g = torch.Generator(device='cuda').manual_seed(1)
    q = torch.randint(-127, 128, (N, K), generator=g, device='cuda', dtype=torch.int8)
    sw = torch.rand(N, generator=g, device='cuda')
    for M in (3, 24):
        x = torch.randn((M, K), generator=g, device='cuda')
        y = P.i8_gemm(P.I8Rows(q, sw, K), x).cpu()
        for a in (0, N - 200):
            assert same(y[:, a:a + 200].contiguous(), product(*rows_of(x.cpu()), q[a:a + 200].cpu().numpy(), sw[a:a + 200].cpu().numpy(), torch.float32))
    del q
    M, N, K = 16500, 140001, 32
    x, w = inputs(M, 1, K, 3)[0], torch.randn((N, K), generator=gen(4))
    y = P.i8_gemm(P.i8_quantize(w.cuda()), x.cuda(), dtype=torch.bfloat16)
    for a in (0, M - 5):
        assert same(y[a:a + 5], product(*rows_of(x[a:a + 5]), *rows_of(w), torch.bfloat16))


# ---- how it is called ----------------------------------------------------------------------------

@pytest.mark.parametrize('M', [1, 4, 12, 140])
def test_captured_replayed_and_on_another_stream(M):
    """Two graphs that share weights and scratch, replayed in turn on another stream with new inputs."""
    P = pkg()
    x, w = inputs(M, 500, 1024, M)
    W, ws = P.i8_quantize(w.cuda()), P.i8_gemm_workspace(M, 1024, 'cuda')
    xs, ys = [x.cuda(), (2 * x).cuda()], [torch.empty((M, 500), device='cuda') for _ in range(2)]
    P.i8_gemm(W, xs[0], ys[0], ws)
    graphs = []
    for a, b in zip(xs, ys):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            P.i8_gemm(W, a, b, ws)
        graphs.append(g)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for seed in (11, 12):
            new = [inputs(M, 1, 1024, seed + i)[0] for i in range(2)]
            for a, n in zip(xs, new):
                a.copy_(n)
            for g in graphs:
                g.replay()
            s.synchronize()
            for n, b in zip(new, ys):
                assert same(b, product(*rows_of(n), *rows_of(w), torch.float32))


@pytest.mark.parametrize('M', [1, 5, 8, 16, 100, 300])
def test_inputs_that_a_kernel_before_writes_late(M):
    """Activations, weights and scales written by a kernel that has released its dependents early."""
    P = pkg()
    x, w = inputs(M, 700, 1536, M)
    W, want = P.i8_quantize(w.cuda()), product(*rows_of(x), *rows_of(w), torch.float32)
    xd, ws, y = x.cuda(), P.i8_gemm_workspace(M, 1536, 'cuda'), torch.empty((M, 700), device='cuda')
    for late in (xd, W.q, W.scale):
        new = late.clone()
        for _ in range(3):
            late.zero_()
            P.i8_gemm(W, xd, y, ws)
            late_copy(late, new)
            P.i8_gemm(W, xd, y, ws)
            assert same(y, want)
    X = P.i8_quantize(xd)
    for late in (X.q, X.scale):
        new = late.clone()
        late.zero_()
        late_copy(late, new)
        P.i8_gemm(W, X, y)
        assert same(y, want)


def test_two_calls_at_once():
    """Two streams, each with its own scratch and outputs, the weights shared; kernels that hold tensor memory on both."""
    P = pkg()
    x, w = inputs(300, 1500, 1200, 1)
    W = P.i8_quantize(w.cuda())
    for Ma, Mb in ((300, 40), (1, 300), (40, 40), (8, 1)):
        xs = [x[:Ma].cuda(), x[:Mb].cuda()]
        want = [P.i8_gemm(W, a) for a in xs]
        ws, ys = [P.i8_gemm_workspace(a.shape[0], 1200, 'cuda') for a in xs], [torch.empty_like(a) for a in want]
        streams = [torch.cuda.Stream() for _ in xs]
        torch.cuda.synchronize()
        for _ in range(20):
            for a, y, s, st in zip(xs, ys, ws, streams):
                P.i8_gemm(W, a, y, s, stream=st)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(ys, want))
    assert P.device_status() == 0


def test_memory_of_a_call_on_another_stream():
    """A call on a stream that is busy, with scratch and outputs of its own: what the current stream allocates next shares none of it."""
    P = pkg()
    x, w = inputs(300, 500, 1200, 1)
    W, xd, s = P.i8_quantize(w.cuda()), x.cuda(), torch.cuda.Stream()
    want = P.i8_gemm(W, xd)
    sizes = [P.i8_gemm_workspace(300, 1200, 'cuda').nbytes, want.nbytes]
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        torch.cuda._sleep(20_000_000)
    y = P.i8_gemm(W, xd, stream=s)
    P.i8_gemm(W, P.i8_quantize(xd, stream=s), stream=s)
    P.token_logprobs(want, torch.zeros((300, 1), dtype=torch.int32, device='cuda'), 5, stream=s)
    taken = [torch.zeros(n, dtype=torch.uint8, device='cuda') for n in sizes + [300 * 1200, 1200, 6000] for _ in range(3)]
    torch.cuda.synchronize()
    assert same(y, want) and not any(t.any() for t in taken)


def test_memory_of_a_call_on_another_stream_that_the_current_one_still_writes():
    """Tensors of the outputs' sizes, freed while the current stream has still to write them: a call on another stream gets none of them."""
    P = pkg()
    x, w = inputs(300, 500, 1200, 1)
    W, xd, s = P.i8_quantize(w.cuda()), x.cuda(), torch.cuda.Stream()
    want, X = P.i8_gemm(W, xd), P.i8_quantize(xd)
    t = torch.zeros((300, 1), dtype=torch.int32, device='cuda')
    wlp = P.token_logprobs(want, t, 5)
    torch.cuda.synchronize()
    sizes = [o.nbytes for o in (want, X.q, X.scale) + wlp] + [P.i8_gemm_workspace(300, 1200, 'cuda').nbytes]
    old = [torch.zeros(n, dtype=torch.uint8, device='cuda') for n in sizes for _ in range(3)]
    torch.cuda.synchronize()
    torch.cuda._sleep(20_000_000)
    for o in old:
        o.fill_(255)
    del old, o
    y, x8, lp = P.i8_gemm(W, xd, stream=s), P.i8_quantize(xd, stream=s), P.token_logprobs(want, t, 5, stream=s)
    torch.cuda.synchronize()
    assert same(y, want) and torch.equal(x8.q, X.q) and torch.equal(x8.scale, X.scale)
    assert all(torch.equal(a, b) for a, b in zip(lp, wlp))


def test_the_same_rows_as_both_operands():
    P = pkg()
    for M in (1, 6, 50, 200):
        x, _ = inputs(M, 1, 500, M)
        r = P.i8_quantize(x.cuda())
        assert same(P.i8_gemm(r, r), product(*rows_of(x), *rows_of(x), torch.float32))


def test_many_calls_back_to_back_beside_the_other_kernels():
    """Products of every size between NVFP4 products that hold tensor memory too, twice the same bits."""
    P = pkg()
    g = torch.Generator(device='cuda').manual_seed(7)
    Wn = P.quantize((torch.randn((2048, 1024), generator=g, device='cuda') * 0.02).to(torch.bfloat16))
    W = P.i8_quantize((torch.randn((2000, 1024), generator=g, device='cuda') * 0.02).to(torch.bfloat16))
    x = torch.randn((400, 1024), generator=g, device='cuda')
    xb, nws = x.to(torch.bfloat16), P.gemm_bf16_workspace(400, 1024, 'cuda')
    got = []
    for _ in range(2):
        outs = []
        for M in (1, 300, 7, 64, 16, 400, 2, 130):
            outs += [P.gemm(Wn, x[:min(M, 8)]), P.i8_gemm(W, x[:M]), P.gemm_bf16(Wn, xb[:M], ws=nws), P.i8_gemm(W, xb[:M])]
        got.append(outs)
    assert all(torch.equal(a, b) for a, b in zip(*got))
    assert P.device_status() == 0


def test_byte_credit():
    P = pkg()
    W = P.i8_quantize(torch.randn((300, 512), generator=gen(1)).cuda())
    for M in (1, 20, 300):
        with P.ByteCredit() as c:
            P.i8_gemm(W, torch.randn((M, 512), generator=gen(M)).cuda())
        assert c.by_kind == {0: 300 * 512.0}


def test_refusals_on_the_gpu():
    P = pkg()
    W, x = P.i8_quantize(torch.ones((8, 64), device='cuda')), torch.ones((4, 64), device='cuda')
    for bad in (dict(x=torch.ones((4, 48), device='cuda')), dict(y=torch.ones((4, 9), device='cuda')), dict(y=torch.ones((8, 4), device='cuda').T),
                dict(y=torch.ones((4, 8), dtype=torch.float16, device='cuda')), dict(ws=torch.empty(256, dtype=torch.uint8, device='cuda')),
                dict(x=x.cpu()), dict(y=torch.ones((4, 8)))):
        a = dict(x=x, y=None, ws=None)
        a.update(bad)
        with pytest.raises(P.B200Error):
            P.i8_gemm(W, a['x'], a['y'], a['ws'])
    with pytest.raises(P.B200Error):
        P.i8_quantize(x, out=P.I8Rows.empty(4, 65, 'cuda'))
