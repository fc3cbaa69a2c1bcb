"""sample_tokens against the oracle in 64 bits: tokens and kept sets are equal, log-probabilities to one rounding."""

import math

import pytest
import torch

from areal_amd.functional import gather_logprobs, sample_tokens
from oracle import token_ends as O

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
SETTINGS = [
    dict(), dict(temperature=0.7), dict(temperature=0.0), dict(top_k=1), dict(top_k=5), dict(top_k=70, temperature=1.3),
    dict(top_p=0.9), dict(top_p=0.3, temperature=2.0), dict(min_p=0.1), dict(min_p=1.0), dict(top_k=40, top_p=0.8),
    dict(top_k=300, top_p=0.95, min_p=0.02), dict(top_k=9, min_p=0.3), dict(top_p=0.6, min_p=0.2), dict(top_p=0.9999),
]


def check(dev, x, u, settings, gpu_x=None):
    """One call against the oracle. A log-probability is a 64-bit difference rounded once to fp32 (2^-24 of it);
    masses are good to 1e-11."""
    on = lambda s: s.to(dev) if torch.is_tensor(s) else s  # noqa: E731
    got = sample_tokens(x.to(dev) if gpu_x is None else gpu_x, u.to(dev), return_kept=True,
                        **{k: on(v) for k, v in settings.items()})
    tokens, lp, full, kept = O.sample(x, u, **settings)
    assert got.tokens.dtype == torch.int64 and got.logprobs.dtype == torch.float32
    assert torch.equal(got.tokens.cpu(), tokens)
    assert torch.equal(got.kept.cpu(), O.pack_bits(kept))
    for a, b in ((got.logprobs, lp), (got.full_logprobs, full)):
        torch.testing.assert_close(a.cpu().double(), b, rtol=2.0**-24 * 1.001, atol=2e-11, equal_nan=True)
    return got


@pytest.mark.parametrize("settings", SETTINGS, ids=str)
@pytest.mark.parametrize("vocab", [1, 2, 7, 8, 31, 32, 33, 65, 1000, 1023, 1024, 1025, 2500])
@pytest.mark.parametrize("dtype", DTYPES)
def test_settings(dev, dtype, vocab, settings):
    g = torch.Generator().manual_seed(vocab)
    x = (torch.randn(5, vocab, generator=g) * 2.5).to(dtype)
    check(dev, x, torch.rand(5, generator=g), settings)


@pytest.mark.parametrize("settings", SETTINGS, ids=str)
@pytest.mark.parametrize("dtype", DTYPES)
def test_ties(dev, dtype, settings):
    """Rows of a few values: cuts fall among equal logits, of either sign and of both zeros."""
    g = torch.Generator().manual_seed(3)
    x = (torch.randn(4, 1500, generator=g) * 1.5).round().to(dtype)
    x[1] = -x[1].abs() - 1
    x[2] = torch.where(torch.rand(1500, generator=g) < 0.5, -0.0, 0.0)
    x[3] = 0.5
    check(dev, x, torch.rand(4, generator=g), settings)


@pytest.mark.parametrize("dtype", DTYPES)
def test_equal_logits_at_exact_borders(dev, dtype):
    x = torch.full((4, 1000), -3.0, dtype=dtype)
    u = torch.tensor([0.0, 0.5, 0.25, 1 - 2.0**-24])
    assert check(dev, x, u, dict()).tokens.tolist() == [0, 500, 250, 999]
    got = check(dev, x, u, dict(top_p=0.5))  # the first 500
    assert got.tokens.tolist() == [0, 250, 125, 499]
    assert check(dev, x, u, dict(top_k=8)).tokens.tolist() == [0, 4, 2, 7]


# candidates that do not fit the list in LDS: flat rows, ties among them, wide limits
@pytest.mark.parametrize("settings", [
    dict(top_p=0.9), dict(top_k=20000), dict(top_k=30000, top_p=0.5), dict(min_p=0.5), dict(top_k=4096), dict(top_k=4097),
    dict(top_k=25000, top_p=0.97, min_p=0.6),
], ids=str)
@pytest.mark.parametrize("kind", ["flat", "ties", "negative"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_many_candidates(dev, dtype, kind, settings):
    g = torch.Generator().manual_seed(5)
    x = torch.randn(3, 50257, generator=g) * 0.3
    if kind == "ties":
        x = (x * 2).round()
    if kind == "negative":
        x -= 40.0
    check(dev, x.to(dtype), torch.rand(3, generator=g), settings)


@pytest.mark.parametrize("dtype", DTYPES)
def test_settings_by_row(dev, dtype):
    g = torch.Generator().manual_seed(6)
    n, v = 37, 4099
    x = (torch.randn(n, v, generator=g) * 2).to(dtype)
    settings = dict(temperature=torch.rand(n, generator=g) * 1.5, top_k=torch.randint(-2, 200, (n,), generator=g),
                    top_p=torch.rand(n, generator=g) * 1.3, min_p=torch.rand(n, generator=g) * 0.3 - 0.1)
    settings["temperature"][::5] = 0.0
    settings["temperature"][1] = -1.0
    settings["top_p"][2] = -0.5
    settings["temperature"][3] = math.inf  # the limit: all finite logits alike
    settings["top_k"][4] = 1 << 40
    u = torch.rand(n, generator=g)
    # at temperature inf the oracle's (x - top) / inf is -0: weight 1, as here
    check(dev, x, u, settings)
    check(dev, x, u.double(), settings | dict(top_k=settings["top_k"].clamp(max=1 << 30).to(torch.int32)))
    for name in ("temperature", "top_p", "min_p"):
        bad = {k: s.clone() for k, s in settings.items()}
        bad[name][7] = math.nan
        assert check(dev, x, u, bad).tokens[7] == -1


@pytest.mark.parametrize("settings", SETTINGS, ids=str)
@pytest.mark.parametrize("dtype", DTYPES)
def test_masked_and_broken_rows(dev, dtype, settings):
    g = torch.Generator().manual_seed(7)
    lowest = torch.finfo(dtype).min
    x = (torch.randn(12, 3333, generator=g) * 2).to(dtype)
    x[0] = -math.inf                     # nothing left
    x[1, 1:] = -math.inf                 # one
    x[2, :-1] = -math.inf
    x[3, 5:3300] = -math.inf             # whole segments masked
    x[4] = lowest                        # all of the lowest value
    x[5, 3:] = lowest                    # masked by it
    x[6, 100] = math.nan
    x[7, 3332] = math.inf
    x[8, 0], x[8, 1] = math.nan, math.inf
    x[9, 0] = torch.finfo(dtype).max     # one far ahead
    x[10] = -math.inf
    x[10, [50, 2000]] = lowest
    u = torch.rand(12, generator=g)
    u[5] = 0.0
    got = check(dev, x, u, settings)
    assert got.tokens[[0, 6, 7, 8]].eq(-1).all() and got.kept[[0, 6, 7, 8]].eq(0).all()


def test_uniforms_outside_the_range(dev):
    g = torch.Generator().manual_seed(8)
    x = torch.randn(6, 2100, generator=g)
    u = torch.tensor([-1.0, 0.0, 1.0, 2.0, math.nan, math.inf])
    for settings in (dict(), dict(top_k=50), dict(top_p=0.999)):
        check(dev, x, u, settings)


def test_extreme_temperatures(dev):
    g = torch.Generator().manual_seed(9)
    x = torch.randn(4, 1100, generator=g)
    for tau in (1e-300, 1e-30, 1e-3, 1e6, 1e300):
        for settings in (dict(), dict(top_p=0.5), dict(top_k=30), dict(min_p=0.5)):
            check(dev, x, torch.rand(4, generator=g), settings | dict(temperature=tau))


@pytest.mark.parametrize("dtype", DTYPES)
def test_layouts(dev, dtype):
    """Rows of any start and pitch, columns apart, more dimensions, one row, none."""
    g = torch.Generator().manual_seed(10)
    base = (torch.randn(3 * 1301 + 3, generator=g) * 2).to(dtype)
    u = torch.rand(3, generator=g)
    for start in (0, 1, 3):
        view = lambda t: t[start:start + 3 * 1301].view(3, 1301)[:, :1290]  # noqa: E731
        for settings in (dict(), dict(top_k=20, top_p=0.9)):
            check(dev, view(base), u, settings, gpu_x=view(base.to(dev)))
    x = (torch.randn(70, 6, generator=g) * 2).to(dtype)
    check(dev, x.t(), torch.rand(6, generator=g), dict(top_p=0.7), gpu_x=x.to(dev).t())
    x = (torch.randn(2, 3, 500, generator=g) * 2).to(dtype)
    u = torch.rand(2, 3, generator=g)
    got = sample_tokens(x.to(dev), u.to(dev), top_k=torch.full((2, 3), 7, device=dev), return_kept=True)
    tokens, lp, _, kept = O.sample(x.view(6, 500), u.view(6), top_k=7)
    assert got.tokens.shape == (2, 3) and got.kept.shape == (2, 3, 16)
    assert torch.equal(got.tokens.cpu().view(6), tokens) and torch.equal(got.kept.cpu().view(6, 16), O.pack_bits(kept))
    one = sample_tokens(x[0, 0].to(dev), u[0, 0].to(dev), top_k=7)
    assert one.tokens.shape == () and int(one.tokens) == int(tokens[0]) and one.kept is None
    none = sample_tokens(x[:0].to(dev), u[:0].to(dev), top_p=0.5, return_kept=True)
    assert none.tokens.shape == (0, 3) and none.kept.shape == (0, 3, 16)
    # a row repeated without memory of its own
    got = sample_tokens(x[0, :1].to(dev).expand(4, 500), torch.rand(4, generator=g).to(dev), top_k=1)
    assert (got.tokens == x[0, 0].float().argmax().item()).all()


@pytest.mark.parametrize("settings", [dict(), dict(top_p=0.9), dict(top_k=50, top_p=0.95)], ids=str)
def test_large_vocabulary(dev, settings):
    g = torch.Generator().manual_seed(11)
    x = (torch.randn(3, 151936, generator=g) * 3).bfloat16()
    check(dev, x, torch.rand(3, generator=g), settings)


def test_largest_vocabulary(dev):
    v = 1 << 22
    x = torch.zeros(1, v, dtype=torch.bfloat16, device=dev)
    u = torch.tensor([0.75], device=dev)
    assert sample_tokens(x, u).tokens.item() == 3 * v // 4
    got = sample_tokens(x, u, top_p=0.5, return_kept=True)
    assert got.tokens.item() == 3 * v // 8
    assert (got.kept[0, : v // 64] == -1).all() and (got.kept[0, v // 64:] == 0).all()
    got = sample_tokens(x, u, top_k=100000)
    assert got.tokens.item() == 75000
    torch.testing.assert_close(got.logprobs.cpu().double(), torch.tensor([-math.log(100000)]).double(), rtol=2.0**-24, atol=2e-11)


@pytest.mark.parametrize("settings", [dict(), dict(top_p=0.9), dict(top_k=50, top_p=0.95, min_p=0.01)], ids=str)
def test_a_row_does_not_depend_on_the_others(dev, settings):
    g = torch.Generator(device=dev).manual_seed(12)
    x = torch.randn(1500, 2049, generator=g, device=dev).bfloat16()
    u = torch.rand(1500, generator=g, device=dev)
    whole = sample_tokens(x, u, return_kept=True, **settings)
    again = sample_tokens(x, u, return_kept=True, **settings)
    for a, b in zip(whole, again):
        assert torch.equal(a, b)
    for i in (0, 777, 1499):
        for a, b in zip(whole, sample_tokens(x[i:i + 1], u[i:i + 1], return_kept=True, **settings)):
            assert torch.equal(a[i:i + 1], b)


@pytest.mark.parametrize("settings", [dict(top_p=0.9), dict(top_p=0.98, temperature=1.5), dict(top_k=30000), dict(min_p=0.2)],
                         ids=str)
@pytest.mark.parametrize("dtype", DTYPES)
def test_wide_rows_in_calls_of_any_size(dev, dtype, settings):
    """Sets of thousands of logits, few of a segment's or nearly all of them, by one row's workgroup of either size or by several."""
    g = torch.Generator(device=dev).manual_seed(15)
    n, v = 300, 100277
    x = torch.randn(n, v, generator=g, device=dev) * 1.8
    x[1::4] = torch.rand(len(x[1::4]), v, generator=g, device=dev) * 0.5
    part = torch.arange(v, device=dev) // 700
    x[2::4] = torch.where(part % 3 == 0, x[1::4], x[2::4] - 6.0)   # segments of one kind and the other
    x[3::4] = x[3::4].sort(1).values                                 # rising
    x[7] = (x[7] * 4).round() / 4                                    # thousands of ties
    x = x.to(dtype)
    u = torch.rand(n, generator=g, device=dev)
    whole = sample_tokens(x, u, return_kept=True, **settings)
    for lo, hi in ((0, 1), (1, 2), (2, 3), (7, 8), (0, 20), (100, 200)):
        got = sample_tokens(x[lo:hi], u[lo:hi], return_kept=True, **settings)
        assert torch.equal(got.tokens, whole.tokens[lo:hi]) and torch.equal(got.kept, whole.kept[lo:hi])
        # sums of masses in another order: 2^-24 and an error of 1e-11 each
        torch.testing.assert_close(got.logprobs, whole.logprobs[lo:hi], rtol=2.0**-23 * 1.001, atol=4e-11)
    rows = [0, 1, 2, 3, 7]
    check(dev, x[rows].cpu(), u[rows].cpu(), settings)
    got = sample_tokens(x, u, return_kept=True, **settings)
    assert torch.equal(got.tokens, whole.tokens) and torch.equal(got.kept, whole.kept)


def test_full_logprobs_are_the_trainers(dev):
    """What the trainer computes for the drawn tokens: fp32 sums of exponents up to ~30 binades (2^-24 each)."""
    g = torch.Generator(device=dev).manual_seed(13)
    x = (torch.randn(64, 32000, generator=g, device=dev) * 3).bfloat16()
    got = sample_tokens(x, torch.rand(64, generator=g, device=dev), temperature=0.8, top_p=0.95)
    torch.testing.assert_close(gather_logprobs(x, got.tokens, 0.8), got.full_logprobs, rtol=1e-6, atol=2e-5)


def test_streams_and_graphs(dev):
    """Inputs of another stream, two graphs of different sizes, replayed in turn with eager calls between."""
    g = torch.Generator(device=dev).manual_seed(14)
    xs = [(torch.randn(n, 5003, generator=g, device=dev) * 2).bfloat16() for n in (3, 50)]
    us = [torch.rand(n, generator=g, device=dev) for n in (3, 50)]
    settings = dict(temperature=0.9, top_k=30, top_p=0.9, return_kept=True)
    want = [sample_tokens(x, u, **settings) for x, u in zip(xs, us)]
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        got = [sample_tokens(x, u, **settings) for x, u in zip(xs, us)]
    torch.cuda.current_stream(dev).wait_stream(side)
    for a, b in zip(want, got):
        assert all(torch.equal(p, q) for p, q in zip(a, b))
    graphs, outs = [], []
    for x, u in zip(xs, us):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(sample_tokens(x, u, **settings))
        graphs.append(graph)
    for _ in range(3):
        for u in us:
            u.copy_(torch.rand(u.shape, generator=g, device=dev))
        want = [sample_tokens(x, u, **settings) for x, u in zip(xs, us)]
        torch.cuda.synchronize()
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(want, outs):
            assert all(torch.equal(p, q) for p, q in zip(a, b))
