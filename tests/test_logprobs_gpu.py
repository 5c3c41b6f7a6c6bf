"""Log probabilities, entropy and best alternatives against 64-bit arithmetic."""
import math

import pytest
import torch

from lightcompress_amd.logprobs import token_logprobs
from tests.helpers import gen

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
INF, LOWEST = float('inf'), torch.finfo(torch.float32).min
U = 2.0 ** -24


def best(x, k):
    """Ids of the k largest of each row: by value, then the lowest id; a NaN first."""
    v = x.double()
    v = torch.where(torch.isnan(v), torch.full_like(v, 1e300), v.clamp(-1e299, 1e299))
    v = torch.where(x == -INF, torch.full_like(v, -1e300), v)
    return torch.sort(v, dim=1, descending=True, stable=True).indices[:, :k]


def check(x, tokens=None, top=0, ignore=-100, got=None):
    """x [T, V].  How far fp32 may be: the sum of V positive terms, at most V / 256 + 64 of them added one after another (a lane's, then
    over lanes and parts), each exp off by 2^-22 and by the rounding of x - c, and a sum whose reference c is up to 8 below the maximum;
    log S itself, x - c and the difference are rounded once more each."""
    got = token_logprobs(x, tokens, top, ignore) if got is None else got
    V = x.shape[1]
    d = x.double()
    logp = torch.log_softmax(d, 1)                  # (less the maximum first: exact also far from zero)
    p = logp.exp()
    H = -torch.where(p == 0, torch.zeros_like(p), p * logp).sum(1)
    A = (V / 256 + 64) * U + 2.0 ** -21
    size = lambda v: torch.where(torch.isfinite(v), v.abs(), torch.zeros_like(v))  # noqa: E731
    tol = lambda v: A + 4 * U * (size(v) + 8 + math.log(V))  # noqa: E731

    def same(a, want, allowed, what):
        a = a.double()
        fine = torch.isfinite(want)
        assert torch.equal(torch.isnan(a), torch.isnan(want)) and torch.equal(a == -INF, want == -INF) and torch.equal(a == INF, want == INF), what
        err = (a - want).abs()[fine]
        assert bool((err <= allowed[fine]).all()), f'{what}: {float((err / allowed[fine]).max())} of the tolerance'

    same(got.entropy, H, 2 * A * (10 + size(H)), 'entropy')
    if tokens is not None:
        t = tokens.reshape(x.shape[0], -1)
        want = logp.gather(1, t.clamp(0, V - 1))
        want = torch.where((t < 0) | (t >= V), torch.full_like(want, math.nan), want)
        want = torch.where(t == ignore, torch.zeros_like(want), want)
        same(got.logprobs.reshape(want.shape), want, tol(want), 'logprobs')
    assert got.top_tokens.shape == (*x.shape[:-1], top)
    ids = best(x, top)
    assert torch.equal(got.top_tokens, ids)
    same(got.top_logprobs, logp.gather(1, ids), tol(logp.gather(1, ids)), 'top')
    return got


@pytest.mark.parametrize('dtype', [BF, HF, F32])
@pytest.mark.parametrize('T,V,top', [(1, 1, 1), (1, 2, 2), (3, 7, 3), (2, 63, 20), (5, 64, 64), (4, 100, 1), (2, 511, 5), (3, 512, 64), (700, 513, 5),
                                     (1, 2047, 10), (2, 2048, 0), (1, 32000, 20), (9, 32001, 64), (1, 128256, 20), (33, 50257, 5), (600, 8191, 2),
                                     (1, 160001, 64), (2048, 1000, 3), (4097, 130, 1), (1100, 70001, 7), (300, 70001, 20), (2, 262144, 64)])
def test_logprobs(dev, T, V, top, dtype):
    x = (torch.randn(T, V, generator=gen(T + V)) * 3).to(dtype).to(dev)
    tokens = torch.randint(0, V, (T,), generator=gen(V)).to(dev)
    check(x, tokens, top)


@pytest.mark.parametrize('T,V', [(1, 5000), (3, 40001), (700, 5000)])
@pytest.mark.parametrize('dtype', [BF, F32])
def test_rows_that_are_special(dev, T, V, dtype):
    """Every kind of row among ordinary ones: its own answer, and the others keep theirs."""
    low = float(torch.finfo(dtype).min)
    rows = torch.randn(12, V, generator=gen(1))
    rows[0] = -INF                                            # nothing left
    rows[1] = low                                             # a mask of the type's lowest value, everywhere
    rows[2, 17] = math.nan
    rows[3, V - 1] = INF
    rows[4] = 2.5                                             # ties everywhere
    rows[5] = -INF
    rows[5, V // 2] = -3.0                                    # one left
    rows[6] = torch.linspace(-50, 50, V)                      # every logit above all before it
    rows[7] = torch.linspace(50, -50, V)
    rows[8, :V - 3] = -INF
    rows[9, 5:] = low
    rows[10] = rows[10] * 1e-3 + 300.0                        # far from zero
    rows[11, ::2] = 0.0
    rows[11, 1::2] = -0.0                                     # equal numbers
    rows = rows.to(dtype)
    pick = torch.arange(max(T, 12)) % 12
    x = rows[pick].to(dev)
    tokens = torch.randint(0, V, (x.shape[0],), generator=gen(2)).to(dev)
    tokens[5] = V // 2
    for top in (0, 1, 20, 64):
        for part in ([slice(0, None)] if T > 12 else [slice(i, i + T) for i in range(0, 12, T)]):
            check(x[part], tokens[part], top)


def test_infinities_of_fp16_and_large_logits(dev):
    x = torch.randn(4, 3001, generator=gen(4))
    x[1] *= 1e30
    x[2] = x[2] * 1e4 + 6e4
    x[3] = -3e38 + 1e37 * x[3]
    check(x.to(dev), torch.arange(4, device=dev), 5)
    h = (torch.randn(2, 3001, generator=gen(5)) * 2e4).to(HF)
    check(h.to(dev), torch.arange(2, device=dev), 5)


def test_given_tokens(dev):
    x = torch.randn(5, 300, generator=gen(6)).to(BF).to(dev)
    t = torch.tensor([0, 299, -100, 300, -1], device=dev)
    got = check(x, t)
    assert float(got.logprobs[2]) == 0.0 and bool(torch.isnan(got.logprobs[3:]).all())
    many = torch.randint(0, 300, (5, 7), generator=gen(7)).to(dev)
    many[1, 2] = 17
    got = check(x, many, ignore=17)
    assert got.logprobs.shape == (5, 7) and bool((got.logprobs[many == 17] == 0).all())
    assert token_logprobs(x).logprobs is None
    assert token_logprobs(x, many[:, :0]).logprobs.shape == (5, 0)


def test_shapes_strides_and_alignment(dev):
    wide = torch.randn(6, 1100, generator=gen(8))
    for dtype in (BF, F32):
        w = wide.to(dtype).to(dev)
        for view in (w[:, :1000], w[:, 1:1001], w[::2, 3:70], w[:, 5:6], w[:1].expand(4, 1100), w.t()[:900].t()):
            a, b = token_logprobs(view, top=1), token_logprobs(view.clone(memory_format=torch.contiguous_format), top=1)
            assert torch.equal(a.top_tokens, b.top_tokens)
            check(view, torch.zeros(view.shape[0], dtype=torch.int64, device=dev), 1, got=None)
        cube = token_logprobs(w.view(2, 3, 1100), torch.zeros(2, 3, dtype=torch.int64, device=dev), top=2)
        flat = token_logprobs(w, torch.zeros(6, dtype=torch.int64, device=dev), top=2)
        assert torch.equal(cube.logprobs.view(-1), flat.logprobs) and torch.equal(cube.top_tokens.view(6, 2), flat.top_tokens)
        assert token_logprobs(w[0], torch.tensor(3, device=dev)).logprobs.shape == ()
    assert token_logprobs(wide[:0].to(dev), top=3).top_tokens.shape == (0, 3)


def test_sequences_without_their_last_logits(dev):
    """logits[:, :-1] next to tokens[:, 1:], as perplexity takes them: the same bits as from a copy."""
    x = (torch.randn(3, 9, 1001, generator=gen(12)) * 3).to(BF).to(dev)
    t = torch.randint(0, 1001, (3, 9), generator=gen(13)).to(dev)
    views = [(x[:, :-1], t[:, 1:]), (x[1:, 2:7], t[1:, :5]), (x[:1, :-1], t[:1, 1:]), (x.transpose(0, 1), t.t()), (x[:, :0], t[:, :0]),
             (x[..., 3:900], t.clamp(max=800)), (x.view(3, 3, 3, 1001)[:, :2, 1:], t.view(3, 3, 3)[:, :2, 1:])]
    for v, ids in views:
        a, b = token_logprobs(v, ids, top=3), token_logprobs(v.clone(memory_format=torch.contiguous_format), ids.clone(), top=3)
        assert all(torch.equal(p, q) and p.shape == q.shape for p, q in zip(a, b))
    x2 = torch.randn(5, 100, 70, generator=gen(14)).to(dev).transpose(0, 1)     # more sequences than are worth a call each
    a, b = token_logprobs(x2, top=2), token_logprobs(x2.contiguous(), top=2)
    assert all(torch.equal(p, q) and p.shape == q.shape for p, q in zip(a[1:], b[1:]))
    a = token_logprobs(x[:, :-1], torch.stack([t[:, 1:], t[:, :-1]], -1))
    want = torch.log_softmax(x[:, :-1].double(), -1).gather(-1, torch.stack([t[:, 1:], t[:, :-1]], -1))
    assert float((a.logprobs - want).abs().max()) < 1e-5


@pytest.mark.parametrize('T,V', [(2, 30000), (700, 30000), (1500, 5000)])
@pytest.mark.parametrize('dtype', [BF, F32])
def test_rows_with_more_ties_than_room(dev, T, V, dtype):
    """Alternatives out of hundreds of equal logits, and of fewer logits than alternatives."""
    x = torch.randn(T, V, generator=gen(T + V))
    x[0] = torch.randint(0, 3, (V,), generator=gen(20)).float()
    x[1] = -INF
    x[1, torch.randint(0, V, (7,), generator=gen(21))] = 1.0
    x[T - 1, ::2] = 9.0
    x[T // 2, V // 3:V // 3 + 513] = 8.0
    for top in (1, 7, 20, 64):
        check(x.to(dtype).to(dev), torch.zeros(T, dtype=torch.int64, device=dev), top)


def test_behind_two_to_the_31(dev):
    T, V = 17000, 128256
    x = torch.zeros(T, V, dtype=BF, device=dev)
    x[-3:] = (torch.randn(3, V, generator=gen(9)) * 3).to(BF).to(dev)
    t = torch.full((T,), 7, dtype=torch.int64, device=dev)
    got = token_logprobs(x, t, top=3)
    check(x[-3:], t[-3:], 3, got=type(got)(*(v[-3:] for v in got)))
    assert bool((got.top_tokens[:-3] == torch.arange(3, device=dev)).all())


def test_more_rows_than_a_launch(dev):
    T, V = 2 ** 21 + 300, 40
    x = torch.randn(T, V, device=dev)
    t = torch.randint(0, V, (T,), device=dev)
    rows = torch.cat([torch.arange(300), 2 ** 21 + torch.arange(-200, 300)]).to(dev)
    got = token_logprobs(x, t, 3)
    check(x[rows], t[rows], 3, got=type(got)(*(v[rows] for v in got)))


def test_captured_and_again(dev):
    """One row (several parts and a join) and many, captured; the same bits on every replay and on every call."""
    xs = [(torch.randn(T, V, generator=gen(T)) * 3).to(BF).to(dev) for T, V in ((1, 50001), (3, 128256), (600, 4000))]
    ids = [torch.zeros(x.shape[0], dtype=torch.int64, device=dev) for x in xs]
    run = lambda: [v for x, t in zip(xs, ids) for v in token_logprobs(x, t, top=8)]  # noqa: E731
    run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for rep in range(3):
        for x in xs:
            x.mul_(0.5 + rep)
        want, again = run(), run()
        torch.cuda.synchronize()
        for o in out:
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(want, out, again)), rep
