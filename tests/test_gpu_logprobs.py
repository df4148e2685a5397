"""Log probabilities of given tokens, entropy and top alternatives against the formulas in 64 bits.

Tolerances.  S = sum exp(x - m) without the likeliest token's 1 is a sum of positive f32 terms: a thread adds at most
n = V / 512 + 64 of them (a term of the sum carries at most 2^-22 of the exponential and |d| 2^-24 ln 2 of its argument, d <= 216,
where the larger arguments weigh least: exp(-d) d < 1), and the joins add 30 roundings.  So S and T are within
r = (n + 100) 2^-24 of their values, relative, and
    ln p          is off by at most r S / (1 + S) <= r, and a rounding each of x - m, ln S and their difference;
    ln p of the likeliest token alone at its value, -log1p(S), by r relative, and log1pf's 2 ulp
    the entropy   by r (ln S + |T| / S) <= 2 r H + 4 roundings of H."""
import numpy as np
import pytest
import torch

from util import pkg
from test_gpu_early_start import late_copy

pytestmark = pytest.mark.gpu
INF = float('inf')


def oracle(x, tokens, top):
    x = x.double().cpu().numpy()
    M, V = x.shape
    bad = ~(x < INF).all(1)
    none = (x == -INF).all(1)
    ok = ~(bad | none)
    xs = np.where(ok[:, None], x, 0.0)
    m = xs.max(1, keepdims=True)
    with np.errstate(all='ignore'):
        d = xs - m
        e = np.exp(d)
        rest = e.sum(1) - 1.0 if V == 1 else np.array([np.delete(r, r.argmax()).sum() for r in e])
        ln_s = np.log1p(rest)                                 # 1 + rest, kept apart as the definition allows
        lp = d - ln_s[:, None]
        h = ln_s - np.where(e > 0, e * np.where(np.isfinite(d), d, 0), 0).sum(1) / (1 + rest)
    lp[none], h[none] = -INF, 0.0
    lp[bad], h[bad] = np.nan, np.nan
    t = tokens.cpu().numpy()
    given = np.where(t < 0, 0.0, np.where(t >= V, np.nan, np.take_along_axis(lp, np.clip(t, 0, V - 1), 1)))
    order = np.stack([np.lexsort((np.arange(V), -r)) if not b else np.arange(V) for r, b in zip(x, bad)])[:, :top]
    ids = np.where(bad[:, None], -1, order)
    return given, h, ids, np.take_along_axis(lp, order, 1), ln_s


def close(got, want, tol):
    got, want = got.cpu().double().numpy(), np.asarray(want)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    inf = np.isinf(want)
    assert np.array_equal(got[inf], want[inf])
    fin = np.isfinite(want)
    assert np.all(np.abs(got - want)[fin] <= np.broadcast_to(tol, want.shape)[fin]), np.max((np.abs(got - want) / tol)[fin])


def check(x, tokens, top, out=None):
    P = pkg()
    xd = x if x.is_cuda else x.cuda()
    td = tokens.cuda()
    lp, h, ids, tlp = P.token_logprobs(xd, td, top, out=out)
    wlp, wh, wids, wtlp, ln_s = oracle(x, tokens, top)
    eps = 2.0 ** -24
    r = (x.shape[1] / 512 + 164) * eps
    scale = np.nan_to_num(np.abs(ln_s), nan=0.0, posinf=0.0)[:, None]
    # S / (1 + S) = 1 - exp(-ln(1 + S)), which double precision loses for S < 2^-53 unless it is taken as -expm1: r S is due there
    tol = lambda w: r * -np.expm1(-scale) + 4 * eps * (2 * np.where(np.isfinite(w), np.abs(w), 0) + 2 * scale) + 1e-38
    close(lp, wlp, tol(wlp))
    close(tlp, wtlp, tol(wtlp))
    close(h, wh, 2 * r * np.where(np.isfinite(wh), wh, 0) + 4 * eps * np.where(np.isfinite(wh), wh, 0) + 1e-38)
    assert np.array_equal(ids.cpu().numpy(), wids)
    return lp, h, ids, tlp


def make(M, V, seed, dtype=torch.float32, sd=2.5):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn((M, V), generator=g) * sd).to(dtype)
    return x, torch.randint(0, V, (M, 3), generator=g, dtype=torch.int32)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('M,V,top', [(1, 1, 1), (2, 2, 1), (3, 7, 7), (1, 9, 0), (5, 31, 31), (4, 100, 32), (2, 255, 20), (3, 513, 32), (1, 2047, 5), (2, 4097, 1),
                                     (1, 8191, 20), (9, 8200, 32), (3, 16390, 20), (1, 32771, 32), (1, 50257, 0), (7, 50257, 20), (40, 20001, 5), (80, 9999, 32),
                                     (150, 4099, 20), (300, 5000, 3), (1, 154880, 20), (5, 154880, 32)])
def test_against_the_formula(M, V, top, dtype):
    x, t = make(M, V, M * V + top, dtype)
    check(x, t, top)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('M,V,top', [(593, 32768, 5), (600, 1000, 32), (700, 20011, 20), (1200, 77, 0), (900, 4099, 1), (640, 2048, 8), (2000, 33, 32)])
def test_many_rows(M, V, top, dtype):
    """Rows enough for the smallest blocks, whole and under masks that leave a row little or nothing.  A thread of 128 adds V / 256 terms to
    each of its two sums, 128 at most, where `check` allows for V / 512 + 164."""
    x, t = make(M, V, M + V, dtype)
    check(x, t, top)
    g = torch.Generator().manual_seed(V)
    x[torch.rand((M, V), generator=g) < 0.97] = -INF
    x[1], x[2], x[3, V // 2], x[4, V - 1] = -INF, torch.finfo(dtype).min, float('nan'), INF
    x[M - 1] = 2.5
    check(x, t, top)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('off,pad', [(0, 0), (1, 0), (3, 5), (2, 1), (5, 3), (8, 47)])
def test_strides_and_alignments(dtype, off, pad):
    M, V = 11, 20011
    x, t = make(M, V, off + pad, dtype)
    big = torch.full((M * (V + pad) + off + 64,), INF, dtype=dtype)
    big = big.cuda()
    view = torch.as_strided(big, (M, V), (V + pad, 1), off)
    view.copy_(x)
    check(view, t, 20)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('V,M', [(300, 3), (20000, 2), (154880, 1), (33333, 40)])
def test_masks(V, M, dtype):
    """-inf and the type's lowest value over most of a row, over all of it, over all but one token, and over the row's first part."""
    P = pkg()
    low = torch.finfo(dtype).min
    for fill in (-INF, low):
        x, t = make(M, V, V + M, dtype)
        g = torch.Generator().manual_seed(5)
        x[torch.rand((M, V), generator=g) < 0.95] = fill
        check(x, t, min(V, 32))
        x[:] = fill
        check(x, t, 5)
        x[0, V - 2] = 1.5
        check(x, t, 5)
        x, t = make(M, V, V, dtype)
        x[:, :V // 2] = fill
        check(x, t, 20)
    x, t = make(M, V, V, dtype)
    x[:, ::2], x[:, 1::4] = -INF, low
    check(x, t, 32)


@pytest.mark.parametrize('fill', [-1e4, -65504.0, -1e9, -1e30, -3.3895313892515355e38])
@pytest.mark.parametrize('V,M', [(20000, 2), (154880, 1), (33333, 600)])
def test_masks_of_other_values(V, M, fill):
    """A mask of some large negative value, over whole rows but for a few tokens and over their first half, beside -inf and smaller values."""
    x, t = make(M, V, M, sd=3.0)
    g = torch.Generator().manual_seed(7)
    keep = torch.rand((M, V), generator=g) < 40.0 / V
    y = torch.where(keep, x, torch.tensor(fill))
    check(y, t, 32)
    check(y.to(torch.bfloat16), t, 20)
    y[:, ::3] = -INF
    check(y, t, 32)
    y[:, 1::7] = 2 * fill if fill > -1e38 else fill
    check(y, t, 20)
    x[:, :V // 2] = fill
    check(x, t, 20)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('V', [1, 40, 5001, 100003])
def test_infinities_and_nan(V, dtype):
    x, t = make(8, V, V, dtype)
    x[0, V - 1] = INF
    x[1, V // 2] = float('nan')
    x[2, 0] = float('nan')
    x[3, :] = -INF
    x[3, V // 3] = float('nan')
    x[4, :] = -INF
    x[4, V - 1] = INF
    x[5, :] = INF
    x[6, :] = -INF
    t[7, 0], t[7, 1], t[0, 0], t[6, 0] = -1, V, -100, -5
    check(x, t, min(V, 6))


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('M', [1, 3, 200])
def test_ties_and_orders(M, dtype):
    """Equal logits throughout, two values, both zeros, ascending and descending rows: what overflows the list of candidates, too."""
    V = 60007
    t = torch.arange(2 * M, dtype=torch.int32).view(M, 2) * 97 % V
    x = torch.full((M, V), 1.25).to(dtype)
    check(x, t, 32)
    x[:, 1::2] = 1.5
    check(x, t, 32)
    x[:, :] = 0.0
    x[:, 3::3] = -0.0
    check(x, t, 20)
    up = torch.linspace(-20, 10, V).to(dtype)
    check(up.expand(M, V).contiguous(), t, 32)
    check(up.flip(0).expand(M, V).contiguous(), t, 32)
    x = up.expand(M, V).contiguous()
    x[:, V - 1] = x[:, V - 3]
    x[:, 0] = x[:, V - 3]
    check(x, t, 7)
    x[:, :] = -3.0
    x[:, V - 1], x[:, 30000] = 2.0, 2.0                                  # the likeliest tie: the last element and one in the middle
    check(x, t, 3)


def test_nearly_certain_tokens_keep_their_precision():
    P = pkg()
    V = 50000
    for gap in (12.0, 17.0, 25.0, 60.0, 110.0):
        x, _ = make(2, V, int(gap), sd=0.5)
        x[:, 777] = gap
        t = torch.full((2, 1), 777, dtype=torch.int32)
        lp, h, ids, tlp = check(x, t, 2)
        w = oracle(x, t, 2)
        r = (V / 512 + 164 + 8) * 2.0 ** -24
        if gap < 80:
            assert np.all(np.abs(lp.cpu().double().numpy() / w[0] - 1) <= r)
            assert np.all(np.abs(h.cpu().double().numpy() / w[1] - 1) <= 2 * r)


@pytest.mark.parametrize('scale', [1e-30, 1.0, 1e4, 1e30, 2e37])
def test_magnitudes(scale):
    x, t = make(3, 3001, 8)
    check(x * scale, t, 9)


def test_no_given_tokens_and_many():
    x, t = make(3, 9000, 1)
    check(x, t[:, :0], 4)
    t = torch.randint(-2, 9003, (3, 1500), generator=torch.Generator().manual_seed(1), dtype=torch.int32)
    check(x, t, 0)


def test_outputs_behind_the_last_stay_and_runs_agree():
    P = pkg()
    x, t = make(37, 30000, 2, torch.bfloat16)
    bufs = [torch.full((40, 3), 7.0, device='cuda'), torch.full((40,), 7.0, device='cuda'), torch.full((40, 20), 7, dtype=torch.int32, device='cuda'),
            torch.full((40, 20), 7.0, device='cuda')]
    first = [o.clone() for o in check(x, t, 20, out=tuple(b[:37] for b in bufs))]
    assert all((b[37:] == 7).all() for b in bufs)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, P.token_logprobs(x.cuda(), t.cuda(), 20)))


def test_a_row_does_not_depend_on_where_it_lies_in_order():
    """Batches whose rows are split alike give a row the same bits."""
    P = pkg()
    x, t = make(37, 30000, 3)
    a = P.token_logprobs(x.cuda(), t.cuda(), 5)
    b = P.token_logprobs(x.flip(0).contiguous().cuda(), t.flip(0).contiguous().cuda(), 5)
    assert all(torch.equal(p, q.flip(0)) for p, q in zip(a, b))


def test_offsets_past_32_bits():
    V, M = 154880, 14001
    x = torch.zeros((M, V), dtype=torch.bfloat16, device='cuda')
    g = torch.Generator(device='cuda').manual_seed(1)
    tail = torch.randn((3, V), generator=g, device='cuda').to(torch.bfloat16)
    x[-3:] = tail
    t = torch.full((M, 1), 5, dtype=torch.int32, device='cuda')
    got = pkg().token_logprobs(x, t, 20)
    want = oracle(tail, t[-3:], 20)
    assert np.array_equal(got[2][-3:].cpu().numpy(), want[2])
    assert np.allclose(got[0][-3:].cpu().numpy(), want[0], rtol=1e-5) and np.allclose(got[1].cpu().numpy()[:4], np.log(V), rtol=1e-5)


@pytest.mark.parametrize('M', [1, 30, 400])
def test_captured_replayed_on_another_stream_and_written_late(M):
    P = pkg()
    x, t = make(M, 12345, M, torch.bfloat16)
    xd, td = x.cuda(), t.cuda()
    out = P.token_logprobs_out(td, 9)
    P.token_logprobs(xd, td, 9, out=out)
    want = [o.clone() for o in out]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        P.token_logprobs(xd, td, 9, out=out)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        for o in out:
            o.zero_()
        g.replay()
        s.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
    torch.cuda.synchronize()
    if M * 12345 % 2 == 0:                                                # the late writer copies whole words
        new = xd.clone()
        xd.zero_()
        P.token_logprobs(xd, td, 9, out=out)
        late_copy(xd, new)
        P.token_logprobs(xd, td, 9, out=out)
        assert all(torch.equal(a, b) for a, b in zip(out, want))
    new = td.clone()
    td.zero_()
    late_copy(td, new)
    P.token_logprobs(xd, td, 9, out=out)
    assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_two_calls_at_once():
    """Two streams, each with its own outputs, again and again: the calls share nothing."""
    P = pkg()
    a, ta = make(40, 30001, 1)
    b, tb = make(3, 154880, 2, torch.bfloat16)
    work = [(a.cuda(), ta.cuda(), 7), (b.cuda(), tb.cuda(), 20)]
    want = [[o.clone() for o in P.token_logprobs(*w)] for w in work]
    outs = [P.token_logprobs_out(w[1], w[2]) for w in work]
    streams = [torch.cuda.Stream() for _ in work]
    torch.cuda.synchronize()
    for _ in range(20):
        for w, o, s in zip(work, outs, streams):
            P.token_logprobs(*w, out=o, stream=s)
    torch.cuda.synchronize()
    for w, o in zip(want, outs):
        assert all(torch.equal(p, q) for p, q in zip(w, o))


@pytest.mark.parametrize('M,V,top', [(1, 154880, 5), (3, 154880, 32), (20, 70001, 20), (37, 50257, 0), (70, 40000, 3)])
def test_rows_shared_by_clusters_beside_busy_multiprocessors(M, V, top):
    """Rows that several CTAs share, while products of another stream take and leave the places that those CTAs start on."""
    P = pkg()
    x, t = make(M, V, M + top)
    xd, td = x.cuda(), t.cuda()
    want = [o.clone() for o in check(x, t, top)]
    g = torch.Generator(device='cuda').manual_seed(3)
    W = P.i8_quantize((torch.randn((3000, 1024), generator=g, device='cuda') * 0.02).to(torch.bfloat16))
    rows = [P.i8_quantize(torch.randn((n, 1024), generator=g, device='cuda')) for n in (2, 30, 300)]
    ys, outs = [torch.empty((r.N, 3000), device='cuda') for r in rows], [P.token_logprobs_out(td, top) for _ in range(30)]
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for o in outs:
        for r, y in zip(rows, ys):
            P.i8_gemm(W, r, y, stream=a)
        P.token_logprobs(xd, td, top, out=o, stream=b)
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for o in outs for p, q in zip(o, want))
    assert P.device_status() == 0


def test_scoring_path_from_hidden_rows():
    """As a scorer runs them: hidden rows -> 8-bit vocabulary projection -> log probabilities, greedy choice and perplexity."""
    P = pkg()
    g = torch.Generator(device='cuda').manual_seed(9)
    M, K, V = 33, 512, 20005
    h = torch.randn((M, K), generator=g, device='cuda').to(torch.bfloat16)
    W = P.i8_quantize((torch.randn((V, K), generator=g, device='cuda') * 0.2).to(torch.bfloat16))
    t = torch.randint(0, V, (M, 1), generator=g, device='cuda', dtype=torch.int32)
    logits = P.i8_gemm(W, h)
    lp, ent, ids, tlp = check(logits, t, 4)
    one = P.token_logprobs(P.i8_gemm(W, h[7:8]), t[7:8], 4)              # a row on its own: the same logits bit for bit
    assert torch.equal(P.i8_gemm(W, h[7:8]), logits[7:8]) and torch.equal(one[2], ids[7:8])
    assert torch.equal(ids[:, 0].long(), logits.argmax(1))
    ppl = float(torch.exp(-lp.double().mean()))
    want = float(torch.exp(-torch.log_softmax(logits.double(), 1).gather(1, t.long()).mean()))
    assert abs(ppl / want - 1) < 1e-5
    assert P.device_status() == 0
