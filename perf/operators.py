"""What is measured of the operators that run a w8a8 model and read its answers.

Four kinds of work, one per step of such a model:

  linear       a w8a8 Linear on floating-point activations: they are quantized per token, multiplied with the int8
               weight and scaled (what VllmRealQuantLinear.forward does)
  matmul       the product alone, of codes that are there already
  norm         the end of one block and the start of the next: [norm], [gate], residual scale, residual, norm
  norm_linear  the same with int8 codes for output, and the Linear that takes them
  logprobs     log probabilities of given tokens, entropy and top alternatives from a model's logits

`run` computes them in elementary torch operations in 32 bits where `own` is false and through the library where it is
true; `exact` has the definitions in 64 bits.
"""
import math

import torch

own = False

DTYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32}
SIZE = {'bf16': 2, 'fp16': 2, 'fp32': 4}
EPS = 1e-5
IGNORED = -100


def listed():
    return [
        # one new token through an attention output projection: latency, and the weight's bytes
        dict(name='linear_1_token', kind='linear', tokens=1, cols=4096, rows=4096, dtype='bf16', asym=False, bias=False),
        # a decode batch of 16 sequences through a down projection, asymmetric activations, a bias
        dict(name='linear_16_tokens_asym', kind='linear', tokens=16, cols=14336, rows=4096, dtype='fp16', asym=True, bias=True),
        # a ragged batch of short prompts through an up projection
        dict(name='linear_211_tokens', kind='linear', tokens=211, cols=4096, rows=14336, dtype='bf16', asym=False, bias=False),
        # a prefill of 8192 tokens through an up projection: the matrix pipe
        dict(name='linear_prefill', kind='linear', tokens=8192, cols=4096, rows=14336, dtype='bf16', asym=False, bias=False),
        # the product alone at sizes that divide by nothing, full-precision output
        dict(name='matmul_odd', kind='matmul', tokens=1333, cols=2047, rows=1001, dtype='fp32', asym=True, bias=True),
        # the norm between two blocks for one new token
        dict(name='norm_1_token', kind='norm', tokens=1, cols=4096, dtype='bf16', norm='rms', post=False, gate=False, scale=1.0, offset=0.0),
        # a long prefill between two blocks, with norms on both sides, gate and residual scale
        dict(name='norm_prefill_gated', kind='norm', tokens=16384, cols=4096, dtype='bf16', norm='rms', post=True, gate=True, scale=0.5, offset=1.0),
        # layer norms in full precision at an odd width
        dict(name='norm_layer_odd', kind='norm', tokens=2049, cols=5121, dtype='fp32', norm='layer', post=True, gate=False, scale=1.0, offset=0.0),
        # the start of an attention block in a prefill: residual, norm, int8 codes, the joint q/k/v projection
        dict(name='norm_linear_qkv', kind='norm_linear', tokens=2048, cols=4096, rows=6144, dtype='bf16', post=False, gate=False, scale=1.0),
        # the next token's alternatives for one sequence
        dict(name='logprobs_1_row', kind='logprobs', tokens=1, vocab=128256, dtype='bf16', top=20, masked=False),
        # perplexity of a 2048-token window, with the five best alternatives
        dict(name='logprobs_window', kind='logprobs', tokens=2048, vocab=128256, dtype='bf16', top=5, masked=False),
        # full-precision logits of a ragged batch with an odd vocabulary, some of it masked out
        dict(name='logprobs_masked', kind='logprobs', tokens=333, vocab=50001, dtype='fp32', top=10, masked=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """Most widths of models are round, some are odd."""
    n = _log(rng, lo, hi)
    return n if rng.random() < 0.3 else max(64, n // 64 * 64)


def draw(rng):
    kind = rng.choice(['linear', 'linear', 'matmul', 'norm', 'norm_linear', 'logprobs'])
    c = dict(kind=kind, dtype=rng.choice(['bf16', 'fp16']))
    if kind in ('linear', 'matmul', 'norm_linear'):
        c.update(tokens=_log(rng, 1, 8192), cols=_width(rng, 256, 14336), rows=_width(rng, 256, 14336))
        while c['tokens'] * c['cols'] * c['rows'] > 8192 * 4096 * 14336:
            c['tokens'] = max(1, c['tokens'] // 2)
    if kind in ('linear', 'matmul'):
        c.update(asym=rng.random() < 0.4, bias=rng.random() < 0.4)
    if kind == 'matmul':
        c['dtype'] = rng.choice(['bf16', 'fp16', 'fp32'])
    if kind == 'norm_linear':
        c.update(post=rng.random() < 0.5, gate=rng.random() < 0.5, scale=rng.choice([1.0, 0.25]))
    if kind == 'norm':
        c.update(tokens=_log(rng, 1, 16384), cols=_width(rng, 64, 14336), dtype=rng.choice(['bf16', 'fp16', 'fp32']),
                 norm=rng.choice(['rms', 'rms', 'layer']), post=rng.random() < 0.5, gate=rng.random() < 0.5,
                 scale=rng.choice([1.0, 0.25]), offset=rng.choice([0.0, 1.0]))
        while c['tokens'] * c['cols'] > 16384 * 4096:
            c['tokens'] = max(1, c['tokens'] // 2)
    if kind == 'logprobs':
        c.update(tokens=_log(rng, 1, 2048), vocab=_width(rng, 1000, 160000), dtype=rng.choice(['bf16', 'fp16', 'fp32']),
                 top=rng.choice([0, 1, 5, 20]), masked=rng.random() < 0.5)
        while c['tokens'] * c['vocab'] * SIZE[c['dtype']] > 2048 * 128256 * 2:
            c['tokens'] = max(1, c['tokens'] // 2)
    return c


# -- inputs -------------------------------------------------------------------------------------------------------
def _activations(tokens, cols, dtype, g):
    """Gaussian with a lognormal scale per channel: outlier channels, as in front of the Linears of a language model."""
    sigma = torch.exp(0.7 * torch.randn(cols, generator=g, device='cuda'))
    return (torch.randn(tokens, cols, generator=g, device='cuda') * sigma).to(DTYPES[dtype])


def _weight(rows, cols, g):
    """An int8 weight with a bf16 scale per channel, as a w8a8 container holds it."""
    w = torch.randn(rows, cols, generator=g, device='cuda') * 0.02
    s = (w.abs().amax(1, keepdim=True).clamp_min(1e-5) / 127).bfloat16()
    return (w / s.float()).round_().clamp_(-128, 127).to(torch.int8), s


def prepare(case, seed):
    c = case
    g = torch.Generator(device='cuda')
    g.manual_seed(seed)
    st = dict(case=c)
    kind = c['kind']
    if kind in ('linear', 'matmul', 'norm_linear'):
        st['w'], st['ws'] = _weight(c['rows'], c['cols'], g)
        st['bias'] = torch.randn(c['rows'], generator=g, device='cuda').to(DTYPES[c['dtype']]) if c.get('bias') else None
    if kind == 'linear':
        st['x'] = _activations(c['tokens'], c['cols'], c['dtype'], g)
        if c['asym']:
            st['x'] += 0.5
    if kind == 'matmul':
        st['codes'] = torch.randn(c['tokens'], c['cols'], generator=g, device='cuda').mul_(32).round_().clamp_(-128, 127).to(torch.int8)
        st['scales'] = 0.01 + 0.05 * torch.rand(c['tokens'], 1, generator=g, device='cuda')
        st['zeros'] = torch.randint(-60, 60, (c['tokens'], 1), generator=g, device='cuda', dtype=torch.int32) if c['asym'] else None
    if kind in ('norm', 'norm_linear'):
        dt = DTYPES[c['dtype']]
        st['x'] = _activations(c['tokens'], c['cols'], c['dtype'], g)
        st['residual'] = _activations(c['tokens'], c['cols'], c['dtype'], g)
        affine = lambda mean: (mean + 0.2 * torch.randn(c['cols'], generator=g, device='cuda')).to(dt)  # noqa: E731
        one = 1.0 - c.get('offset', 0.0)
        st['weight'] = affine(one)
        st['post_weight'] = affine(one) if c['post'] else None
        layer = c.get('norm') == 'layer'
        st['norm_bias'] = affine(0.0) if layer else None
        st['post_bias'] = affine(0.0) if layer and c['post'] else None
        st['gate'] = torch.sigmoid(torch.randn(c['tokens'], c['cols'], generator=g, device='cuda')).to(dt) if c['gate'] else None
    if kind == 'logprobs':
        T, V = c['tokens'], c['vocab']
        x = torch.randn(T, V, generator=g, device='cuda').mul_(2.5)
        picked = torch.randint(0, V, (T, 1), generator=g, device='cuda')
        x.scatter_add_(1, picked, 12 * torch.rand(T, 1, generator=g, device='cuda'))      # a model that knows something
        other = torch.randint(0, V, (T, 1), generator=g, device='cuda')
        tokens = torch.where(torch.rand(T, 1, generator=g, device='cuda') < 0.5, picked, other)
        if c['masked']:
            x[:, V - V // 50:] = -math.inf                                               # padded vocabulary
            x.masked_fill_(torch.rand(1, V, generator=g, device='cuda') < 0.1, -math.inf)  # a grammar's mask
            x.scatter_(1, tokens, 1.5)                                                   # (the given tokens are allowed)
            tokens = tokens.masked_fill(torch.rand(T, 1, generator=g, device='cuda') < 0.1, IGNORED)  # padding
        st['logits'], st['tokens'] = x.to(DTYPES[c['dtype']]), tokens[:, 0].contiguous()
    return st


# -- the plain forms ----------------------------------------------------------------------------------------------
def _codes(x, asym):
    """x [T, K] in 32 bits -> codes, scales, zero points, the first and last as 32-bit floats."""
    if not asym:
        s = x.abs().amax(1, keepdim=True).clamp_min(1e-5) / 127
        return torch.round(x / s).clamp_(-128, 127), s, None
    lo, hi = x.amin(1, keepdim=True), x.amax(1, keepdim=True)
    s = (hi - lo).clamp_min(1e-5) / 255
    z = (-128 - torch.round(lo / s)).clamp(-128, 127)
    return (torch.round(x / s) + z).clamp_(-128, 127), s, z


def _product(q, s, z, st, dtype):
    if z is not None:
        q = q - z
    y = (q @ st['w'].float().t()) * s * st['ws'].float().t()
    if st['bias'] is not None:
        y = y + st['bias'].float()
    return y.to(dtype)


def _norm(x, kind, weight, bias, offset):
    if kind == 'layer':
        x = x - x.mean(1, keepdim=True)
    y = x * torch.rsqrt(x.square().mean(1, keepdim=True) + EPS) * (weight.float() + offset)
    return y if bias is None else y + bias.float()


def _residual_norm(st):
    c = st['case']
    kind, offset = c.get('norm', 'rms'), c.get('offset', 0.0)
    b = st['x'].float()
    if c['post']:
        b = _norm(b, kind, st['post_weight'], st['post_bias'], offset)
    if c['gate']:
        b = b * st['gate'].float()
    h = st['residual'].float() + c['scale'] * b
    return h, _norm(h, kind, st['weight'], st['norm_bias'], offset)


def _logprobs(st):
    c, tokens = st['case'], st['tokens'][:, None]
    x = st['logits'].float()
    m = x.amax(1, keepdim=True)
    e = torch.exp(x - m)
    total = e.sum(1, keepdim=True)
    lse = m + torch.log(total)
    given = tokens != IGNORED
    logp = torch.where(given, x.gather(1, tokens.clamp_min(0)) - lse, 0.0)
    entropy = lse - torch.where(e > 0, e * x, 0.0).sum(1, keepdim=True) / total
    out = dict(logprobs=logp[:, 0], entropy=entropy[:, 0])
    if c['top']:
        # one whole number per logit that orders by value and then by the lowest index
        bits = (x + 0.0).view(torch.int32)
        key = torch.where(bits < 0, bits ^ 0x7fffffff, bits).to(torch.int64) * (1 << 32) - torch.arange(c['vocab'], device=x.device)
        at = (-torch.topk(key, c['top'], dim=1).values) & 0xffffffff
        out.update(top_logprobs=x.gather(1, at) - lse, top_tokens=at)
    return out


def _plain(st):
    c = st['case']
    kind, dt = c['kind'], DTYPES[c['dtype']]
    if kind == 'linear':
        return _product(*_codes(st['x'].float(), c['asym']), st, dt)
    if kind == 'matmul':
        return _product(st['codes'].float(), st['scales'], None if st['zeros'] is None else st['zeros'].float(), st, dt)
    if kind == 'logprobs':
        return _logprobs(st)
    h, y = _residual_norm(st)
    if kind == 'norm':
        return dict(residual=h.to(dt), out=y.to(dt))
    return dict(residual=h.to(dt), out=_product(*_codes(y, False), st, dt))


# -- the library's calls ------------------------------------------------------------------------------------------
def _own(st):
    from lightcompress_amd.logprobs import token_logprobs
    from lightcompress_amd.w8a8 import QuantizedTokens, int8_linear, int8_matmul, residual_norm
    c = st['case']
    kind, dt = c['kind'], DTYPES[c['dtype']]
    if kind == 'linear':
        return int8_linear(st['x'], st['w'], st['ws'], st['bias'], symmetric=not c['asym'])
    if kind == 'matmul':
        return int8_matmul(QuantizedTokens(st['codes'], st['scales'], st['zeros']), st['w'], st['ws'], st['bias'], out_dtype=dt)
    if kind == 'logprobs':
        r = token_logprobs(st['logits'], st['tokens'], top=c['top'], ignore_index=IGNORED)
        out = dict(logprobs=r.logprobs, entropy=r.entropy)
        if c['top']:
            out.update(top_logprobs=r.top_logprobs, top_tokens=r.top_tokens)
        return out
    r = residual_norm(st['x'], st['residual'], st['weight'], st['norm_bias'], gate=st['gate'], post_weight=st['post_weight'],
                      post_bias=st['post_bias'], scale=c['scale'], eps=EPS, kind=c.get('norm', 'rms'),
                      weight_offset=c.get('offset', 0.0), quantize='symmetric' if kind == 'norm_linear' else None)
    if kind == 'norm':
        return dict(residual=r.residual, out=r.out)
    return dict(residual=r.residual, out=int8_matmul(r.out, st['w'], st['ws'], out_dtype=dt))


def run(state):
    return _own(state) if own else _plain(state)


# -- the definitions in 64 bits -----------------------------------------------------------------------------------
def exact(case, seed):
    st, c = prepare(case, seed), case
    f = torch.float64

    def linear(v, asym):
        """v [T, K] in 64 bits; a token's scale is a 32-bit number by definition."""
        top = v.amax(1) if asym else torch.maximum(v.amax(1), -v.amin(1))
        low = v.amin(1) if asym else torch.zeros_like(top)
        s = ((top - low).clamp(min=1e-5) / (255 if asym else 127)).float().to(f)[:, None]
        z = (-128 - torch.round(low[:, None] / s)).clamp(-128, 127) if asym else torch.zeros_like(s)
        q = torch.clamp(torch.round(v / s) + z, -128, 127)
        return scaled(q - z, s)

    def scaled(q, s):
        y = torch.mm(q, st['w'].to(f).t()) * (s * st['ws'].to(f).view(1, -1))
        return y if st['bias'] is None else y + st['bias'].to(f)

    def normed(v, w, b):
        if c.get('norm', 'rms') == 'layer':
            var, mean = torch.var_mean(v, dim=1, correction=0, keepdim=True)
            v = (v - mean) / torch.sqrt(var + EPS)
        else:
            v = v / torch.sqrt((v * v).mean(1, keepdim=True) + EPS)
        v = v * (w.to(f) + c.get('offset', 0.0))
        return v if b is None else v + b.to(f)

    if c['kind'] == 'linear':
        return linear(st['x'].to(f), c['asym'])
    if c['kind'] == 'matmul':
        q = st['codes'].to(f)
        return scaled(q if st['zeros'] is None else q - st['zeros'].to(f), st['scales'].to(f))
    if c['kind'] in ('norm', 'norm_linear'):
        b = st['x'].to(f)
        if st['post_weight'] is not None:
            b = normed(b, st['post_weight'], st['post_bias'])
        if st['gate'] is not None:
            b = st['gate'].to(f) * b
        h = b * c['scale'] + st['residual'].to(f)
        y = normed(h, st['weight'], st['norm_bias'])
        return dict(residual=h, out=y if c['kind'] == 'norm' else linear(y, False))
    x = st['logits'].to(f)
    logp = x - torch.logsumexp(x, 1, keepdim=True)
    p = torch.exp(logp)
    entropy = -torch.where(p > 0, p * logp, torch.zeros((), dtype=f, device=x.device)).sum(1)
    kept = st['tokens'] != IGNORED
    at = torch.where(kept, st['tokens'], 0)
    out = dict(logprobs=torch.where(kept, logp[torch.arange(x.shape[0], device=x.device), at], 0.0), entropy=entropy)
    if c['top']:
        out.update(top_logprobs=torch.topk(logp, c['top'], dim=1).values, top_tokens=None)
    return out


def work(case):
    c, b = case, SIZE[case['dtype']]
    T = c['tokens']
    if c['kind'] == 'logprobs':
        V, k = c['vocab'], c['top']
        return dict(bytes=T * V * b + T * (8 + 4 + 4 + 12 * k), flops=6 * T * V)
    K = c['cols']
    if c['kind'] in ('norm', 'norm_linear'):
        read = T * K * b * (3 if c['gate'] else 2) + K * b
        if c['kind'] == 'norm':
            return dict(bytes=read + 2 * T * K * b, flops=10 * T * K)
        N = c['rows']
        return dict(bytes=read + T * K * b + N * K + 2 * N + T * N * b, flops=2 * T * N * K + 12 * T * K)
    N = c['rows']
    a = T * K * (1 if c['kind'] == 'matmul' else b)
    return dict(bytes=a + N * K + 2 * N + T * N * b + (N * b if c['bias'] else 0), flops=2 * T * N * K)
