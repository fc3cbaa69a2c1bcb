"""gather_kept_logprobs_entropy, forward and backward, against the oracle in 64 bits."""

import math

import pytest
import torch

from areal_amd.functional import gather_kept_logprobs_entropy, gather_logprobs_entropy
from oracle import token_ends as O

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def tolerance(x, tau):
    """An exponent x / tau in base 2 is off by the rounding of 1 / tau, of its product with log2(e), of that with x and of
    the row's maximum, 2^-24 of its size each; differences of two of them and the exponential (1 ulp) enter a
    probability, a logarithm and a sum of them: at most 16 such errors of the largest exponent."""
    top = x[torch.isfinite(x)].abs().max().double().item() / tau if torch.isfinite(x).any() else 0.0
    return 16 * 2.0**-24 * (1.0 + min(top, 1e3))


def check(dev, x, labels, mask, tau=1.0, gpu_x=None, words=None, grads=None):
    g = torch.Generator().manual_seed(1)
    n = x.shape[0]
    glp, gent = grads if grads else (torch.randn(n, generator=g), torch.randn(n, generator=g))
    xg = (x.to(dev) if gpu_x is None else gpu_x).detach().requires_grad_(True)
    words = O.pack_bits(mask).to(dev) if words is None else words
    lp, ent = gather_kept_logprobs_entropy(xg, labels.to(dev), words, tau)
    want_lp, want_ent = O.kept_logprobs_entropy(x, labels, mask, tau)
    tol = tolerance(x[mask], tau)
    torch.testing.assert_close(lp.detach().cpu().double(), want_lp, rtol=2.0**-22, atol=tol, equal_nan=True)
    # the entropy is a sum of p log p with log p up to the range of the exponents
    spread = 1 + tolerance(x[mask], tau) * 2.0**20
    torch.testing.assert_close(ent.detach().cpu().double(), want_ent, rtol=2.0**-20, atol=tol * spread, equal_nan=True)
    for use_lp, use_ent in ((True, True), (True, False), (False, True)):
        outs = [o for o, use in ((lp, use_lp), (ent, use_ent)) if use]
        ups = [w.to(dev) for w, use in ((glp, use_lp), (gent, use_ent)) if use]
        (d,) = torch.autograd.grad(outs, xg, ups, retain_graph=True)
        assert d.dtype == x.dtype and d.shape == x.shape
        want = O.kept_backward(x, labels, mask, glp * use_lp, gent * use_ent, tau)
        half_step = torch.finfo(x.dtype).eps / 2
        tiny = torch.finfo(x.dtype).smallest_normal * 2.0**-10
        torch.testing.assert_close(d.cpu().double(), want, rtol=half_step + 2.0**-20,
                                   atol=tol * spread * 8 / tau + tiny, equal_nan=True)
        assert (d.cpu()[~mask] == 0).all()
    return lp, ent, xg


@pytest.mark.parametrize("tau", [1.0, 0.7])
@pytest.mark.parametrize("share", [0.02, 0.5, 1.0])
@pytest.mark.parametrize("vocab", [1, 7, 8, 31, 32, 33, 65, 2047, 2048, 2049, 5003, 9000])
@pytest.mark.parametrize("dtype", DTYPES)
def test_sizes(dev, dtype, vocab, share, tau):
    g = torch.Generator().manual_seed(vocab)
    n = 6
    x = (torch.randn(n, vocab, generator=g) * 2).to(dtype)
    mask = torch.rand(n, vocab, generator=g) < share
    labels = torch.randint(0, vocab, (n,), generator=g)
    mask[torch.arange(n), labels] = True
    mask[1] = False            # nothing kept
    mask[2, labels[2]] = False  # the label not kept
    labels[3] = -100           # an ignored position
    labels[4] = vocab
    check(dev, x, labels, mask, tau)


@pytest.mark.parametrize("rows", [1, 1023, 1024, 1025])
def test_row_counts(dev, rows):
    g = torch.Generator().manual_seed(rows)
    x = torch.randn(rows, 300, generator=g).bfloat16()
    mask = torch.rand(rows, 300, generator=g) < 0.3
    check(dev, x, torch.randint(0, 300, (rows,), generator=g), mask, 0.9)


@pytest.mark.parametrize("dtype", DTYPES)
def test_masked_places_do_not_matter(dev, dtype):
    g = torch.Generator().manual_seed(2)
    n, v = 8, 4500
    x = (torch.randn(n, v, generator=g) * 2).to(dtype)
    mask = torch.rand(n, v, generator=g) < 0.2
    labels = torch.tensor([int(torch.nonzero(m)[3]) for m in mask])
    clean = x.clone()
    lp0, ent0, xg = check(dev, x, labels, mask, 0.9)
    (d0,) = torch.autograd.grad((lp0, ent0), xg, (torch.ones(n, device=dev), torch.ones(n, device=dev)))
    for value in (math.nan, math.inf, -math.inf, torch.finfo(dtype).max, torch.finfo(dtype).min):
        x = clean.masked_fill(~mask, value)
        lp, ent, xg = check(dev, x, labels, mask, 0.9)
        (d,) = torch.autograd.grad((lp, ent), xg, (torch.ones(n, device=dev), torch.ones(n, device=dev)))
        assert torch.equal(lp, lp0) and torch.equal(ent, ent0) and torch.equal(d, d0)


@pytest.mark.parametrize("dtype", DTYPES)
def test_kept_values_that_are_not_finite(dev, dtype):
    g = torch.Generator().manual_seed(3)
    n, v = 8, 2100
    x = (torch.randn(n, v, generator=g) * 2).to(dtype)
    mask = torch.rand(n, v, generator=g) < 0.1
    labels = torch.tensor([int(torch.nonzero(m)[3]) for m in mask])
    at = lambda r, i: int(torch.nonzero(mask[r])[i])  # noqa: E731
    x[0, at(0, 0)] = math.nan
    x[1, at(1, 5)] = math.inf
    x[2, at(2, 1)] = -math.inf           # adds nothing
    x[3, labels[3]] = -math.inf          # the label's own
    x[4, mask[4]] = -math.inf            # all of them
    x[5, mask[5]] = math.nan
    x[6, at(6, 0)] = torch.finfo(dtype).min
    lp, ent, _ = check(dev, x, labels, mask)
    assert torch.isnan(lp[[0, 1, 5]]).all() and torch.isnan(ent[[0, 1, 5]]).all()
    assert lp[3] == lp[4] == -math.inf and ent[4] == 0


@pytest.mark.parametrize("tau", [1.0, 2.0, 0.5, 1e-38, 1e30])
@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_that_keep_only_lowest_values(dev, dtype, tau):
    """Masking with the type's lowest finite value: a row that keeps nothing else is uniform, not empty."""
    g = torch.Generator().manual_seed(7)
    n, v = 6, 4500
    low, top = torch.finfo(dtype).min, torch.finfo(dtype).max
    x = torch.full((n, v), low, dtype=dtype)
    mask = torch.rand(n, v, generator=g) < 0.3
    mask[0] = True
    labels = torch.tensor([int(torch.nonzero(m)[9]) for m in mask])
    x[1, ~mask[1]] = top                 # not kept
    x[2, labels[2]] = top                # all of the mass (or, in fp16 at the highest temperature, its share)
    alone = (top - low) / tau > 1e3
    x[3, torch.nonzero(mask[3])[50:, 0]] = -math.inf
    x[4, labels[4]] = -math.inf
    mask[5], labels[5] = False, 4499
    mask[5, 4499] = True                 # one, at the end
    count = torch.tensor([v, int(mask[1].sum()), 1 if alone else int(mask[2].sum()), 50, int(mask[4].sum()) - 1, 1]).double()
    glp, gent = torch.randn(n, generator=g), torch.randn(n, generator=g)
    xg = x.to(dev).requires_grad_(True)
    lp, ent = gather_kept_logprobs_entropy(xg, labels.to(dev), O.pack_bits(mask).to(dev), tau)
    # exponents are 0 or below the lowest: one rounding each of the logarithm (2 units), its product and ln 2
    want = -count.log()
    want[4] = -math.inf
    torch.testing.assert_close(lp.detach().cpu().double(), want, rtol=2.0**-21, atol=0)
    torch.testing.assert_close(ent.detach().cpu().double(), count.log(), rtol=2.0**-21, atol=0)
    # p is off by the exponent's rounding (log2 of the count, 13 at most, in 2 units) and the exponential's
    (d,) = torch.autograd.grad(lp, xg, glp.to(dev), retain_graph=True)
    p = (mask & (x > -math.inf)).double() / count[:, None]
    if alone:
        p[2] = 0.0
        p[2, labels[2]] = 1.0
    one = torch.zeros(n, v, dtype=torch.float64).scatter_(1, labels[:, None], 1.0)
    want = glp.double()[:, None] * (one - p) / tau
    want[4] = 0.0
    cap = torch.finfo(dtype).max
    scale = glp.double().abs()[:, None] / tau
    bound = scale * p * 2.0**-18 + scale * one * 2.0**-22 + torch.finfo(dtype).eps / 2 * want.abs()
    bound = bound + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    fits = want.abs() < cap
    off = (d.cpu().double() - want).abs()
    assert (off[fits] <= bound[fits]).all(), (off[fits] - bound[fits]).max()
    # p (log p + entropy) is 0 in a uniform row, up to the errors of both logarithms
    (d,) = torch.autograd.grad(ent, xg, gent.to(dev))
    bound = gent.double().abs()[:, None] / tau * p * (2.0**-18 * (1 + count.log()[:, None]))
    bound = bound + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    # (times 1 / tau = 1e38 the errors alone, 2^-24 and up, are 6e30: out of fp16's range they are rounded to infinity)
    bound = torch.where(bound > cap, math.inf, bound)
    assert (d.cpu().double().abs() <= bound).all()


def test_a_label_of_the_lowest_value(dev):
    x = torch.zeros(2, 40, device=dev)
    x[:, 7] = torch.finfo(torch.float32).min
    x[1, 3] = torch.finfo(torch.float32).max
    xg = x.requires_grad_(True)
    words = torch.full((2, 2), -1, dtype=torch.int32, device=dev)
    lp, ent = gather_kept_logprobs_entropy(xg, torch.tensor([7, 7], device=dev), words)
    assert lp[0] == torch.finfo(torch.float32).min and lp[1] == -math.inf  # -6.8e38 is out of range
    torch.testing.assert_close(ent.detach().cpu(), torch.tensor([math.log(39), 0.0]), rtol=2.0**-21, atol=0)
    (d,) = torch.autograd.grad(lp, xg, torch.ones(2, device=dev))
    torch.testing.assert_close(d[0].cpu(), torch.full((40,), -1 / 39).index_fill_(0, torch.tensor(7), 1.0),
                               rtol=2.0**-18, atol=0)
    assert torch.isfinite(d).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_layouts(dev, dtype):
    """Rows of any start and pitch, more words than the vocabulary needs and bits behind it, more dimensions."""
    g = torch.Generator().manual_seed(4)
    base = (torch.randn(3 * 2111 + 3, generator=g) * 2).to(dtype)
    mask = torch.rand(3, 2103, generator=g) < 0.4
    labels = torch.tensor([0, 2102, 1000])
    wide = torch.full((3, 70), -1, dtype=torch.int32)
    wide[:, :66] = O.pack_bits(mask)
    wide[:, 65] |= -1 << (2103 - 65 * 32)
    for start in (0, 1, 3):
        view = lambda t: t[start:start + 3 * 2111].view(3, 2111)[:, :2103]  # noqa: E731
        check(dev, view(base), labels, mask, 0.8, gpu_x=view(base.to(dev)), words=wide.to(dev))
    x, m = (torch.randn(60, 5, generator=g)).to(dtype), torch.rand(5, 60, generator=g) < 0.5
    check(dev, x.t(), torch.arange(5), m, gpu_x=x.to(dev).t())
    strided = torch.zeros(5, 4, dtype=torch.int32, device=dev)
    strided[:, ::2] = O.pack_bits(m).to(dev)
    check(dev, x.t(), torch.arange(5), m, gpu_x=x.to(dev).t(), words=strided[:, ::2])
    x3 = torch.randn(2, 3, 40, generator=g).to(dtype).to(dev).requires_grad_(True)
    lp, ent = gather_kept_logprobs_entropy(x3, torch.zeros(2, 3, dtype=torch.long, device=dev),
                                           torch.full((2, 3, 2), -1, dtype=torch.int32, device=dev))
    assert lp.shape == ent.shape == (2, 3)
    (lp.sum() + ent.sum()).backward()
    assert x3.grad.shape == (2, 3, 40)
    lp, ent = gather_kept_logprobs_entropy(x3[:0], torch.zeros(0, 3, dtype=torch.long, device=dev),
                                           torch.zeros(0, 3, 2, dtype=torch.int32, device=dev))
    assert lp.shape == (0, 3)
    (lp.sum() + ent.sum()).backward()


def test_all_kept_is_the_plain_softmax(dev):
    g = torch.Generator(device=dev).manual_seed(5)
    x = (torch.randn(40, 50257, generator=g, device=dev) * 2).bfloat16().requires_grad_(True)
    y = torch.randint(0, 50257, (40,), generator=g, device=dev)
    words = torch.full((40, 1571), -1, dtype=torch.int32, device=dev)
    ups = (torch.randn(40, generator=g, device=dev), torch.randn(40, generator=g, device=dev))
    got, want = gather_kept_logprobs_entropy(x, y, words, 0.9), gather_logprobs_entropy(x, y, 0.9)
    for a, b in zip(got, want):
        torch.testing.assert_close(a, b, rtol=2.0**-20, atol=2 * tolerance(x.detach(), 0.9))
    (a,), (b,) = (torch.autograd.grad(o, x, ups) for o in (got, want))
    torch.testing.assert_close(a, b, rtol=2.0**-7, atol=1e-7)  # two roundings of bf16


def test_no_gradient_for_an_upstream_of_minus_infinity(dev):
    """A loss may make a NaN of the -inf of a label that is not kept: that row's log-probability has no gradient."""
    x = torch.randn(2, 100, device=dev, requires_grad=True)
    words = torch.tensor([[1, 0, 0, 0], [3, 0, 0, 0]], dtype=torch.int32, device=dev)
    lp, _ = gather_kept_logprobs_entropy(x, torch.tensor([5, 1], device=dev), words)
    lp.backward(torch.tensor([math.nan, 1.0], device=dev))
    assert (x.grad[0] == 0).all() and (x.grad[1, :2] != 0).all()


def test_no_grad_and_streams_and_graphs(dev):
    g = torch.Generator(device=dev).manual_seed(6)
    x = torch.randn(9, 3001, generator=g, device=dev).requires_grad_(True)
    y = torch.randint(0, 3001, (9,), generator=g, device=dev)
    words = torch.randint(-(1 << 31), 1 << 31, (9, 94), generator=g, device=dev, dtype=torch.int64).to(torch.int32)
    ups = (torch.randn(9, generator=g, device=dev), torch.randn(9, generator=g, device=dev))

    def call():
        outs = gather_kept_logprobs_entropy(x, y, words, 0.9)
        return (*[o.detach() for o in outs], *torch.autograd.grad(outs, x, ups))

    with torch.no_grad():
        lp, _ = gather_kept_logprobs_entropy(x, y, words, 0.9)
    assert not lp.requires_grad and torch.equal(lp, call()[0])
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        other = call()
    torch.cuda.current_stream(dev).wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(call(), other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = call()
    for _ in range(3):
        with torch.no_grad():
            x.copy_(torch.randn(9, 3001, generator=g, device=dev))
        want = call()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, outs))
