"""Products of 8-bit integers and the log probabilities of given tokens, as cases that can be timed and checked.

    own                  False: the operators in plain torch; True: this library's calls
    listed()             the cases, each a dict of plain values
    draw(rng)            one more case of the same ranges
    prepare(case, seed)  what a program holds before the call, on the GPU
    run(state)           one pass through an operator; returns its outputs
    work(case)           bytes and operations the pass cannot do without
    exact(case, seed)    the outputs from the definition, in 64 bits

Two operators.

gemm       y[m, n] = sx[m] * sw[n] * sum_k qx[m, k] * qw[n, k], all q whole numbers in -127 .. 127.  Rows of a matrix are
           brought to that form by one rule, the weights once (a scale per output channel), activations within the call
           (a scale per token): a = max(max |row|, 2^-119), scale = a / 127, q = round_half_even(x * (127 / a)), every
           step one fp32 operation.  `kind: siblings` quantises the tokens once for several products that share them.
logprobs   of logits [rows, vocab]: log p of the given tokens, the entropy of p in nats, and the `top` likeliest tokens
           with their log p, ties to the lowest index.  A masked token has logit -inf.

Sizes: hidden 4096, dense MLP 12288, linear-attention projections of 8192 rows, low-rank ones of 128, vocabulary
154880; others are generic.
"""
import math

import torch

own = False

F32, BF16 = 'f32', 'bf16'
_DT = {F32: torch.float32, BF16: torch.bfloat16}


def listed():
    return [
        # One decode token through a low-rank gate: the smallest product, where only latency counts.
        {'name': 'i8 gemm low rank', 'kind': 'gemm', 'rows': 1, 'hidden': 4096, 'outs': 128, 'x': F32, 'y': F32},
        # One decode token through a projection of the layer's width.
        {'name': 'i8 gemm decode', 'kind': 'gemm', 'rows': 1, 'hidden': 4096, 'outs': 4096, 'x': BF16, 'y': F32},
        # The vocabulary projection of one decode token: the largest weight stream.
        {'name': 'i8 gemm head', 'kind': 'gemm', 'rows': 1, 'hidden': 4096, 'outs': 154880, 'x': F32, 'y': F32},
        # A decode batch of five sequences (an odd batch) through the dense MLP's gate.
        {'name': 'i8 gemm batch 5', 'kind': 'gemm', 'rows': 5, 'hidden': 4096, 'outs': 12288, 'x': BF16, 'y': F32},
        # A decode batch of 24 sequences through the MLP's way back, a long sum.
        {'name': 'i8 gemm batch 24', 'kind': 'gemm', 'rows': 24, 'hidden': 12288, 'outs': 4096, 'x': BF16, 'y': BF16},
        # A short prompt of ragged length through three projections that share their input.
        {'name': 'i8 siblings 301', 'kind': 'siblings', 'rows': 301, 'hidden': 4096, 'outs': 8192, 'n': 3, 'x': BF16, 'y': BF16},
        # A prefill chunk whose sizes are multiples of nothing.
        {'name': 'i8 gemm odd 777', 'kind': 'gemm', 'rows': 777, 'hidden': 2051, 'outs': 5003, 'x': F32, 'y': F32},
        # A full prefill chunk through the dense MLP's gate: bound by the matrix instructions.
        {'name': 'i8 gemm prefill 2048', 'kind': 'gemm', 'rows': 2048, 'hidden': 4096, 'outs': 12288, 'x': BF16, 'y': BF16},
        # The answer's next token, with the alternatives that an API shows.
        {'name': 'logprobs decode', 'kind': 'logprobs', 'rows': 1, 'vocab': 154880, 'pad': 0, 'top': 5, 'given': 1, 'x': F32, 'mask': 0.0},
        # A batch under a grammar that forbids most tokens; an odd vocabulary in rows padded to a multiple of 64.
        {'name': 'logprobs batch 37', 'kind': 'logprobs', 'rows': 37, 'vocab': 50257, 'pad': 47, 'top': 20, 'given': 4, 'x': BF16, 'mask': 0.9},
        # Perplexity over a chunk of text: only the given tokens' log probabilities and the entropy.
        {'name': 'logprobs text 512', 'kind': 'logprobs', 'rows': 512, 'vocab': 154880, 'pad': 0, 'top': 0, 'given': 1, 'x': BF16, 'mask': 0.0},
        # A whole prefill chunk scored, with twenty alternatives for each token: the largest stream of logits.
        {'name': 'logprobs prompt 2048', 'kind': 'logprobs', 'rows': 2048, 'vocab': 154880, 'pad': 0, 'top': 20, 'given': 1, 'x': F32, 'mask': 0.0},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(['gemm', 'gemm', 'gemm', 'siblings', 'logprobs', 'logprobs', 'logprobs'])
    x, y = rng.choice([F32, BF16]), rng.choice([F32, BF16])
    if kind == 'logprobs':
        vocab = _log_int(rng, 100, 154880)
        rows = _log_int(rng, 1, 2048)
        return {'kind': kind, 'rows': rows, 'vocab': vocab, 'pad': rng.choice([0, 0, -vocab % 64]), 'top': rng.choice([0, 1, 5, 20, 32]),
                'given': rng.choice([1, 1, 3, 9]), 'x': x, 'mask': rng.choice([0.0, 0.0, 0.5, 0.99])}
    hidden = rng.choice([_log_int(rng, 64, 12288), 16 * _log_int(rng, 8, 768), 256 * rng.randint(2, 16)])
    if kind == 'siblings':
        return {'kind': kind, 'rows': _log_int(rng, 1, 700), 'hidden': min(hidden, 4096), 'outs': _log_int(rng, 64, 8192), 'n': rng.randint(2, 3),
                'x': x, 'y': y}
    outs = rng.choice([_log_int(rng, 32, 12288), _log_int(rng, 32, 12288), _log_int(rng, 12288, 154880)])
    most = min(2048, 2048 * 12288 * 4096 // (outs * hidden))
    return {'kind': kind, 'rows': min(most, rng.choice([rng.randint(1, 8), rng.randint(9, 64), _log_int(rng, 1, 2048)])), 'hidden': hidden, 'outs': outs,
            'x': x, 'y': y}


# ---- inputs --------------------------------------------------------------------------------------

class _Gen:
    """Seeded device tensors."""

    def __init__(self, seed):
        self.g = torch.Generator(device='cuda').manual_seed(seed)

    def normal(self, *shape):
        return torch.randn(shape, generator=self.g, device='cuda')

    def uniform(self, *shape):
        return torch.rand(shape, generator=self.g, device='cuda')

    def whole(self, below, *shape):
        return torch.randint(0, below, shape, generator=self.g, device='cuda')


def _gemm_inputs(case, seed):
    """Activations [rows, hidden] with a few large channels, the last of several rows a padding row of zeros, and bf16
    weights [outs, hidden] whose channels differ in size."""
    g, M, K, N = _Gen(seed), case['rows'], case['hidden'], case['outs']
    x = g.normal(M, K) * torch.where(g.uniform(K) < 0.002, 12.0, 1.0)
    if M > 1:
        x[-1] = 0.0
    ws = [(g.normal(N, K) * (0.02 * (0.5 + g.uniform(N, 1)))).to(torch.bfloat16) for _ in range(case.get('n', 1))]
    return x.to(_DT[case['x']]), ws


def _logits(case, seed):
    """Logits of a model that is fairly sure of the given tokens, and the given tokens [rows, given] i32."""
    g, M, V, G = _Gen(seed), case['rows'], case['vocab'], case['given']
    full = torch.empty((M, V + case['pad']), dtype=_DT[case['x']], device='cuda')
    tokens = g.whole(V, M, G)
    boost = 6.0 + 4.0 * g.normal(M, 1)
    for a in range(0, M, 256):
        part = g.normal(min(256, M - a), V + case['pad']).mul_(2.5)
        if case['mask']:
            part.masked_fill_(g.uniform(*part.shape) < case['mask'], -math.inf)
        t = tokens[a:a + 256, :1]
        part.scatter_(1, t, boost[a:a + 256])
        full[a:a + 256] = part
    return full[:, :V], tokens.to(torch.int32)


def _package():
    import __graft_entry__
    return __graft_entry__.load_package()


def prepare(case, seed):
    kind = case['kind']
    if kind == 'logprobs':
        x, tokens = _logits(case, seed)
        s = {'kind': kind, 'x': x, 'tokens': tokens, 'top': case['top']}
        if own:
            s['P'] = P = _package()
            s['out'] = P.token_logprobs_out(tokens, case['top'])
        return s
    x, ws = _gemm_inputs(case, seed)
    M, K, N, dt = case['rows'], case['hidden'], case['outs'], _DT[case['y']]
    s = {'kind': kind, 'x': x, 'dt': dt}
    if own:
        s['P'] = P = _package()
        s['W'] = [P.i8_quantize(w) for w in ws]
        s['y'] = [torch.empty((M, N), dtype=dt, device='cuda') for _ in ws]
        s['xq'] = P.I8Rows.empty(M, K, 'cuda') if kind == 'siblings' else None
        s['ws'] = P.i8_gemm_workspace(M, K, 'cuda') if kind == 'gemm' else None
    else:
        s['W'] = [_plain_rows(w) for w in ws]
        s['W'] = [(q.to(torch.int8), scale) for q, scale in s['W']]
    return s


# ---- one pass ------------------------------------------------------------------------------------

def run(s):
    kind = s['kind']
    if not own:
        if kind == 'logprobs':
            return _plain_logprobs(s['x'], s['tokens'], s['top'])
        qx, sx = _plain_rows(s['x'])
        ys = [((qx @ qw.float().T) * sx[:, None] * sw).to(s['dt']) for qw, sw in s['W']]
        return ys if kind == 'siblings' else ys[0]
    P = s['P']
    if kind == 'logprobs':
        return P.token_logprobs(s['x'], s['tokens'], s['top'], out=s['out'])
    if kind == 'gemm':
        return P.i8_gemm(s['W'][0], s['x'], s['y'][0], ws=s['ws'])
    xq = P.i8_quantize(s['x'], out=s['xq'])
    return [P.i8_gemm(W, xq, y) for W, y in zip(s['W'], s['y'])]


def _plain_rows(x):
    """(whole numbers as f32, scale per row).  Products of such rows are whole numbers; the sums of these cases stay below
    2^24, where f32 holds each of them."""
    x = x.float()
    a = x.abs().amax(1).clamp_min(2.0 ** -119)
    most = torch.full_like(a, 127.0)                             # a tensor: torch divides by a plain number through its reciprocal
    return torch.round(x * (most / a)[:, None]), a / most


def _plain_logprobs(x, tokens, top):
    x = x.float()
    m = x.amax(1, keepdim=True)
    d = x - m
    e = torch.exp(d)
    total = e.sum(1, keepdim=True, dtype=torch.float64)          # in 64 bits: log p of a sure token is the log of nearly one
    entropy = total.log() - torch.where(e > 0, e * d, 0.0).sum(1, keepdim=True, dtype=torch.float64) / total
    of = lambda ids: (d.gather(1, ids).double() - total.log()).float()
    # one whole-number key per token: f32 bits in an order that ascends with the value, then the lower index first
    top_ids = torch.empty((x.shape[0], 0), dtype=torch.int64, device=x.device)
    if top:
        bits = (x + 0.0).view(torch.int32).long()                # -0 and +0 are the same logit
        key = torch.where(bits < 0, bits ^ 0x7fffffff, bits) * (1 << 32) - torch.arange(x.shape[1], device=x.device)
        top_ids = torch.topk(key, top, dim=1).indices
    return of(tokens.long()), entropy[:, 0].float(), top_ids.to(torch.int32), of(top_ids)


# ---- what a pass costs, and its outputs in 64 bits -----------------------------------------------

def work(case):
    M, es = case['rows'], 4 if case['x'] == F32 else 2
    if case['kind'] == 'logprobs':
        V, G, top = case['vocab'], case['given'], case['top']
        return {'bytes': M * (V * es + 8 * G + 4 + 8 * top), 'flops': 4 * M * V}       # difference, exponential, two sums
    K, N, n = case['hidden'], case['outs'], case.get('n', 1)
    return {'bytes': n * (N * K + 4 * N) + M * (K * es + n * N * (4 if case['y'] == F32 else 2)), 'flops': 2 * n * M * N * K}


def _exact_rows(x):
    """The rule's fp32 steps, then whole numbers in 64 bits."""
    a = torch.maximum(x.float().abs().max(dim=1).values, torch.tensor(2.0 ** -119, device=x.device))
    # a quotient of two f32 rounded to 64 bits and then to f32 is the f32 quotient: 53 >= 2 * 24 + 2
    inv, scale = (127.0 / a.double()).float(), (a.double() / 127.0).float()
    return (x.float() * inv.unsqueeze(1)).round().double(), scale.double()


def exact(case, seed):
    if case['kind'] == 'logprobs':
        x, tokens = _logits(case, seed)
        parts = []
        for a in range(0, x.shape[0], 64):
            v = x[a:a + 64].double()
            logp = v - torch.logsumexp(v, 1, keepdim=True)
            p = logp.exp()
            order = torch.sort(v, dim=1, descending=True, stable=True).indices[:, :case['top']]
            parts.append((torch.gather(logp, 1, tokens[a:a + 64].long()), torch.special.entr(p).sum(1), order.to(torch.int32),
                          torch.gather(logp, 1, order)))
        return tuple(torch.cat(t) for t in zip(*parts))
    x, ws = _gemm_inputs(case, seed)
    qx, sx = _exact_rows(x)
    out = []
    for w in ws:
        qw, sw = _exact_rows(w)
        out.append(torch.cat([torch.matmul(qx, qw[a:a + 8192].T) * (sx.unsqueeze(1) * sw[a:a + 8192]) for a in range(0, qw.shape[0], 8192)], dim=1))
    return out if case['kind'] == 'siblings' else out[0]
