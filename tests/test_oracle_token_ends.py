"""The oracle of sampling, kept-set log-probabilities and embedding lookup against closed forms, brute
force and differences."""

import math

import pytest
import torch

from oracle import token_ends as O


def test_order_cuts_and_ties():
    x = [1.0, 3.0, 3.0, -math.inf, 2.0, 3.0]
    kept = lambda **s: [i for i, k in enumerate(O.sample_row(x, 0.0, **s)[3]) if k]  # noqa: E731
    assert kept() == [0, 1, 2, 4, 5]
    assert kept(top_k=2) == [1, 2] and kept(top_k=4) == [1, 2, 4, 5] and kept(top_k=99) == [0, 1, 2, 4, 5]
    assert kept(temperature=0.0) == [1] and kept(top_k=1) == [1]
    assert kept(top_p=0.01) == [1]
    # of three equal ones a third of their mass is the first, a little more the first two
    assert kept(top_k=3, top_p=0.33) == [1] and kept(top_k=3, top_p=0.34) == [1, 2]
    assert kept(min_p=0.9) == [1, 2, 5] and kept(min_p=1.0) == [1, 2, 5] and kept(min_p=math.exp(-1.5)) == [1, 2, 4, 5]
    assert O.sample_row([-math.inf] * 3, 0.5)[0] == -1 and O.sample_row([1.0, math.nan], 0.5)[0] == -1
    assert O.sample_row([0.0, math.inf], 0.5)[0] == -1


def test_inversion_gives_the_distribution():
    g = torch.Generator().manual_seed(0)
    x, n = torch.randn(17, generator=g, dtype=torch.float64), 20000
    tokens, lps, fulls, kepts = zip(*[O.sample_row(x.tolist(), (i + 0.5) / n, 0.7, 9, 0.8, 0.05) for i in range(n)])
    kept = torch.tensor(kepts[0])
    z = (x / 0.7).masked_fill(~kept, -math.inf)
    p = torch.softmax(z, 0)
    assert ((torch.bincount(torch.tensor(tokens), minlength=17) / n - p).abs() <= 1.0 / n).all()
    for t, lp, full in zip(tokens[::997], lps[::997], fulls[::997]):
        assert lp == pytest.approx(float(p[t].log()), rel=1e-12)
        assert full == pytest.approx(float(torch.log_softmax(x / 0.7, 0)[t]), rel=1e-12)


def test_bits():
    m = torch.zeros(2, 65, dtype=torch.bool)
    m[0, [0, 31, 32, 64]] = True
    assert O.pack_bits(m).tolist() == [[1 - (1 << 31), 1, 1], [0, 0, 0]]


def test_kept_softmax_and_its_gradient_against_differences():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(5, 11, generator=g, dtype=torch.float64)
    mask = torch.rand(5, 11, generator=g) < 0.6
    mask[3] = False
    mask[4] = True
    labels = torch.tensor([int(torch.nonzero(m)[0]) if m.any() else 2 for m in mask])
    labels[2] = int(torch.nonzero(~mask[2])[0])  # not kept
    lp, ent = O.kept_logprobs_entropy(x, labels, mask, 0.8)
    assert lp[2] == lp[3] == -math.inf and ent[3] == 0
    torch.testing.assert_close(lp[4], torch.log_softmax(x[4] / 0.8, 0)[labels[4]])
    glp, gent = torch.randn(5, generator=g), torch.randn(5, generator=g)
    got = O.kept_backward(x, labels, mask, glp, gent, 0.8)
    assert (got[~mask] == 0).all()
    h = 1e-5
    for j in range(11):
        step = torch.zeros_like(x)
        step[:, j] = h
        (lp1, e1), (lp0, e0) = (O.kept_logprobs_entropy(x + s * step, labels, mask, 0.8) for s in (1, -1))
        dlp = torch.where(torch.isfinite(lp), (lp1 - lp0) / (2 * h), torch.zeros_like(lp))
        want = glp * dlp + gent * (e1 - e0) / (2 * h)
        torch.testing.assert_close(got[:, j], want, rtol=1e-7, atol=1e-8)


def test_embedding_gradient_against_differences():
    g = torch.Generator().manual_seed(2)
    w = torch.randn(7, 3, generator=g, dtype=torch.float64)
    ids = torch.tensor([[1, 6, 1], [-1, 7, 0]])
    grad = torch.randn(2, 3, 3, generator=g, dtype=torch.float64)
    dw, count, _ = O.embedding_backward(grad, ids, (7, 3), 1.5)
    assert count.tolist() == [1, 2, 0, 0, 0, 0, 1]
    for v in range(7):
        for c in range(3):
            step = torch.zeros_like(w)
            step[v, c] = 1.0
            diff = ((O.embedding(w + step, ids, 1.5) - O.embedding(w - step, ids, 1.5)) * grad).sum() / 2
            assert float(dw[v, c]) == pytest.approx(float(diff), abs=1e-12)
    assert (O.embedding_backward(grad, ids, (7, 3), 1.5, padding_idx=1)[0][1] == 0).all()
