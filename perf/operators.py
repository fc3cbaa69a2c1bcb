"""Workloads of the operators at the token ends of a model.

* ``sample``  next tokens from logits, with temperature, top-k, top-p and min-p, from given
  uniform numbers (``functional.sample_tokens``)
* ``kept``    log-probabilities and entropy of labels under the kept sets their tokens were drawn
  from, and their gradient (``functional.gather_kept_logprobs_entropy``)
* ``embed``   rows of the ``[V, H]`` weight for token ids, and the weight's gradient
  (``functional.embed_tokens``)

Where ``own`` is false ``run`` computes them with elementary torch operations. Hidden sizes and
vocabularies are those of ``perf/cases.py``.
"""

from __future__ import annotations

import math

import torch

own = False  # True: ``run`` calls the framework's operators

# (hidden size, vocabulary)
MODELS = [
    (896, 151936), (1024, 151936), (1536, 151936), (2048, 151936), (2560, 151936), (3584, 152064),
    (4096, 128256), (4096, 151936), (5120, 151936), (8192, 128256),
]
VOCABS = [32000, 50257, 128256, 151936, 152064]
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
MAX_SAMPLE = 1024 * 151936     # rows x vocabulary of the largest sampling call
MAX_KEPT = 2048 * 151936       # the same of the largest training call
MAX_EMBED = (32768 * 3 + 151936) * 4096  # values read and written by the largest embedding step


# -- the cases -------------------------------------------------------------------------------

def listed():
    return [
        # One sequence being decoded with the usual generation settings: latency.
        dict(name="sample one row", op="sample", rows=1, vocab=151936, dtype="bf16", filters="both", kept=False),
        # A serving batch whose requests each bring their own settings, greedy ones among them.
        dict(name="sample mixed 64", op="sample", rows=64, vocab=151936, dtype="fp32", filters="rows", kept=False),
        # A rollout batch with top-p whose kept sets go to the trainer.
        dict(name="sample top-p 512 kept", op="sample", rows=512, vocab=128256, dtype="bf16", filters="top_p", kept=True),
        # A rollout batch from the whole distribution, the setting of on-policy training.
        dict(name="sample plain 1024", op="sample", rows=1024, vocab=151936, dtype="bf16", filters="none", kept=False),
        # An odd vocabulary: rows of any alignment, fp16 logits, settings by row, kept sets.
        dict(name="sample ragged 77", op="sample", rows=77, vocab=50257, dtype="fp16", filters="rows", kept=True),
        # The log-probabilities of a short response, odd vocabulary, fp32 logits.
        dict(name="kept ragged 93", op="kept", rows=93, vocab=50257, dtype="fp32", temperature=0.8),
        # A micro-batch of a model that makes its logits: log-probabilities, entropy, gradient.
        dict(name="kept 2048", op="kept", rows=2048, vocab=151936, dtype="bf16", temperature=1.0),
        # The tokens of one decode step.
        dict(name="embed decode 64", op="embed", tokens=64, hidden=4096, vocab=151936, weight="bf16", out="bf16", grad=False),
        # A packed batch that only log-probabilities are wanted of.
        dict(name="embed 32k", op="embed", tokens=32768, hidden=4096, vocab=151936, weight="bf16", out="bf16", grad=False),
        # A short left-over micro-batch of the smallest model: the gradient is nearly all zeros.
        dict(name="embed step 509", op="embed", tokens=509, hidden=896, vocab=151936, weight="bf16", out="bf16", grad=True),
        # Mixed precision: fp32 master weights, bf16 activations, fp32 gradient.
        dict(name="embed step fp32 masters", op="embed", tokens=16384, hidden=1536, vocab=151936, weight="fp32", out="bf16", grad=True),
        # The embedding's share of a large training step.
        dict(name="embed step 32k", op="embed", tokens=32768, hidden=4096, vocab=151936, weight="bf16", out="bf16", grad=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    op = rng.choice(["sample", "sample", "sample", "kept", "embed", "embed"])
    if op == "sample":
        vocab = rng.choice(VOCABS) + rng.choice([0, 0, 1, -3])
        dtype = rng.choice(["bf16", "bf16", "fp32", "fp16"])
        return dict(op=op, rows=_log_int(rng, 1, MAX_SAMPLE * 2 // BYTES[dtype] // vocab), vocab=vocab, dtype=dtype,
                    filters=rng.choice(["none", "both", "top_k", "top_p", "min_p", "rows", "rows"]), kept=rng.random() < 0.4)
    if op == "kept":
        vocab = rng.choice(VOCABS) + rng.choice([0, 0, 1, -3])
        dtype = rng.choice(["bf16", "bf16", "fp32", "fp16"])
        return dict(op=op, rows=_log_int(rng, 8, MAX_KEPT * 2 // BYTES[dtype] // vocab), vocab=vocab, dtype=dtype,
                    temperature=rng.choice([0.6, 0.8, 1.0, 1.2]))
    hidden, vocab = rng.choice(MODELS)
    weight = rng.choice(["bf16", "bf16", "fp32"])
    grad = rng.random() < 0.6 and (4096 * 3 + vocab) * hidden * BYTES[weight] <= MAX_EMBED * 2
    most = (MAX_EMBED * 2 // BYTES[weight] // hidden - vocab) // 3 if grad else 32768
    return dict(op=op, tokens=_log_int(rng, 1, min(32768, most)), hidden=hidden, vocab=vocab, weight=weight,
                out=rng.choice([weight, "bf16"]), grad=grad)


# -- what a case cannot do without ------------------------------------------------------------

def work(case):
    if case["op"] == "sample":  # logits in; token and two log-probabilities, the bits of the kept set out
        n = case["rows"] * case["vocab"]
        return dict(bytes=n * BYTES[case["dtype"]] + (n // 8 if case["kept"] else 0) + 40 * case["rows"], flops=20 * n)
    if case["op"] == "kept":  # the bits, the logits of the rows that keep all; the gradient out
        n = case["rows"] * case["vocab"]
        return dict(bytes=n // 8 + (n + n // 4) * BYTES[case["dtype"]] + 40 * case["rows"], flops=10 * n)
    t, h, v = case["tokens"], case["hidden"], case["vocab"]
    read = len(set(_zipf_rows(t, v)))  # rows of the weight that are read at all
    there = 8 * t + read * h * BYTES[case["weight"]] + t * h * BYTES[case["out"]]
    back = t * h * BYTES[case["out"]] + v * h * BYTES[case["weight"]] if case["grad"] else 0
    return dict(bytes=there + back, flops=(2 if case["grad"] else 1) * t * h)


def _zipf_rows(tokens, vocab):
    """Ids as ``_ids`` draws them, at evenly spaced quantiles."""
    return [int(vocab * ((i + 0.5) / tokens) ** 3) for i in range(tokens)]


# -- inputs -----------------------------------------------------------------------------------

def _device():
    return torch.device("cuda", torch.cuda.current_device())


def _logits(rows, vocab, dtype, g):
    """Logits of rows of different sharpness: a normal body, and a few tokens that stand out."""
    dev = _device()
    spread = 1.5 + 1.5 * torch.rand(rows, 1, generator=g, device=dev)
    x = torch.randn(rows, vocab, generator=g, device=dev) * spread
    heads = torch.randint(0, vocab, (rows, 12), generator=g, device=dev)
    x.scatter_(1, heads, 4.0 * spread + 3.0 * torch.rand(rows, 12, generator=g, device=dev))
    return x.to(dtype)


def _ids(tokens, vocab, g):
    """Token ids, low ones (the frequent tokens of a vocabulary) far more often; the last 3 % are padding, id 0."""
    r = torch.rand(tokens, generator=g, device=_device(), dtype=torch.float64)
    ids = (vocab * r * r * r).long().clamp_(max=vocab - 1)
    ids[tokens - tokens // 32:] = 0
    return ids


def _pack_bits(mask):
    """Bool ``[N, V]`` to int32 words ``[N, ceil(V / 32)]``: bit j of word w is token 32 w + j."""
    n, v = mask.shape
    words = (v + 31) // 32
    out = torch.zeros(n, words, dtype=torch.int64, device=mask.device)
    for j in range(32):
        part = mask[:, j::32]
        out[:, : part.shape[1]] |= part.long() << j
    return torch.where(out >= 1 << 31, out - (1 << 32), out).to(torch.int32)


def prepare(case, seed):
    dev = _device()
    g = torch.Generator(device=dev).manual_seed(seed)
    rand = lambda *shape: torch.rand(*shape, generator=g, device=dev)  # noqa: E731
    s = dict(case)
    if case["op"] == "sample":
        n = case["rows"]
        s["logits"] = _logits(n, case["vocab"], DTYPES[case["dtype"]], g)
        s["uniforms"] = rand(n)
        s["settings"] = {
            "none": dict(temperature=1.0),
            "both": dict(temperature=0.7, top_k=50, top_p=0.95),
            "top_k": dict(temperature=1.0, top_k=200),
            "top_p": dict(temperature=1.0, top_p=0.9),
            "min_p": dict(temperature=1.2, min_p=0.05),
        }.get(case["filters"])
        if case["filters"] == "rows":
            kind = torch.randint(0, 4, (n,), generator=g, device=dev)  # greedy, top-k + top-p, top-p, min-p
            temperature = 0.6 + 0.6 * rand(n)
            top_k = torch.randint(1, 100, (n,), generator=g, device=dev, dtype=torch.int32)
            s["settings"] = dict(
                temperature=torch.where(kind == 0, torch.zeros_like(temperature), temperature),
                top_k=torch.where(kind == 1, top_k, torch.zeros_like(top_k)),
                top_p=torch.where((kind == 1) | (kind == 2), 0.8 + 0.19 * rand(n), torch.ones(n, device=dev)),
                min_p=torch.where(kind == 3, 0.02 + 0.1 * rand(n), torch.zeros(n, device=dev)),
            )
    elif case["op"] == "kept":
        n, v = case["rows"], case["vocab"]
        x = _logits(n, v, DTYPES[case["dtype"]], g)
        # kept sets of the policy that drew the tokens: within a margin of its largest logit, or all (a
        # quarter of the rows); the label is one of them
        old = x.float() + 0.05 * torch.randn(n, v, generator=g, device=dev)
        margin = torch.where(rand(n, 1) < 0.25, torch.full((n, 1), 1e9, device=dev), 1.0 + 5.0 * rand(n, 1))
        mask = old >= old.amax(1, keepdim=True) - margin
        old += -torch.log(-torch.log(rand(n, v).clamp_(1e-7, 1 - 1e-7)))
        s["labels"] = old.masked_fill_(~mask, -math.inf).argmax(1)
        s["kept"] = _pack_bits(mask)
        s["logits"] = x.requires_grad_(True)
        s["grads"] = (torch.randn(n, generator=g, device=dev), 0.01 * torch.randn(n, generator=g, device=dev))
    else:
        t, h, v = case["tokens"], case["hidden"], case["vocab"]
        s["ids"] = _ids(t, v, g)
        w = torch.empty(v, h, device=dev, dtype=DTYPES[case["weight"]]).normal_(0, 0.02, generator=g)
        s["weight"] = w.requires_grad_(case["grad"])
        s["scale"] = math.sqrt(h)
        if case["grad"]:
            s["grad_out"] = torch.empty(t, h, device=dev, dtype=DTYPES[case["out"]]).normal_(0, 1e-3, generator=g)
    return s


# -- the plain forms --------------------------------------------------------------------------

def _row(setting, default, rows, dev):
    """A setting as a [rows, 1] fp64 tensor."""
    if torch.is_tensor(setting):
        return setting.double().view(rows, 1)
    return torch.full((rows, 1), float(default if setting is None else setting), dtype=torch.float64, device=dev)


def _plain_sample(logits, uniforms, settings, with_kept):
    n, v = logits.shape
    x = logits.double()
    tau = _row(settings.get("temperature"), 1.0, n, x.device)
    k = _row(settings.get("top_k"), 0, n, x.device)
    p = _row(settings.get("top_p"), 1.0, n, x.device)
    min_p = _row(settings.get("min_p"), 0.0, n, x.device)
    greedy = tau <= 0
    k = torch.where(greedy, torch.ones_like(k), torch.where(k > 0, k, torch.full_like(k, v)))
    tau = torch.where(greedy, torch.ones_like(tau), tau)
    top = x.amax(1, keepdim=True)
    e = torch.exp((x - top) / tau)
    if any(name in settings for name in ("top_k", "top_p", "min_p")):
        _, order = torch.sort(x, dim=1, descending=True, stable=True)  # ties: the lowest index first
        es = e.gather(1, order)
        rank = torch.arange(v, device=x.device).unsqueeze(0)
        es = torch.where(rank < k, es, torch.zeros_like(es))
        mass = es.cumsum(1)
        keep = (rank < k) & ((mass - es < p * mass[:, -1:]) | (p >= 1)) & (es >= min_p)
        keep[:, 0] = True
        kept = torch.zeros_like(keep).scatter_(1, order, keep)
        del order, es, mass, keep
    else:
        kept = torch.ones_like(x, dtype=torch.bool)
    kept &= x > -math.inf
    weight = torch.where(kept, e, torch.zeros_like(e))
    c = weight.cumsum(1)
    tokens = (c <= uniforms.double().unsqueeze(1) * c[:, -1:]).sum(1)
    last = v - 1 - kept.flip(1).to(torch.uint8).argmax(1)
    tokens = torch.minimum(tokens, last)
    exponent = ((x.gather(1, tokens.unsqueeze(1)) - top) / tau)
    lp = (exponent - torch.log(c[:, -1:])).squeeze(1)
    full = torch.where(greedy, torch.zeros_like(exponent), exponent - torch.log(e.sum(1, keepdim=True))).squeeze(1)
    out = dict(tokens=tokens, logprobs=lp.float(), full_logprobs=full.float())
    if with_kept:
        out["kept"] = _pack_bits(kept)
    return out


def _unpack_bits(words, v):
    bits = (words.unsqueeze(-1) >> torch.arange(32, device=words.device, dtype=torch.int32)) & 1
    return bits.view(words.shape[0], -1)[:, :v].bool()


def _plain_kept(logits, labels, kept, temperature, grad_lp, grad_ent):
    mask = _unpack_bits(kept, logits.shape[1])
    z = logits.detach().float() / temperature
    z = z.masked_fill(~mask, -math.inf)
    z = z - z.amax(1, keepdim=True)
    e = torch.exp(z)
    s = e.sum(1, keepdim=True)
    logp = z - torch.log(s)
    p = e / s
    lp = logp.gather(1, labels.unsqueeze(1)).squeeze(1)
    logp = logp.masked_fill(~mask, 0.0)
    ent = -(p * logp).sum(1)
    d = -p * grad_lp.unsqueeze(1) - grad_ent.unsqueeze(1) * p * (logp + ent.unsqueeze(1))
    d.scatter_add_(1, labels.unsqueeze(1), grad_lp.unsqueeze(1))
    return lp, ent, (d / temperature).to(logits.dtype)


def _plain_embed(ids, weight, scale, out_dtype, grad_out):
    w = weight.detach()
    out = (w[ids].float() * scale).to(out_dtype)
    if grad_out is None:
        return (out,)
    dw = torch.zeros(w.shape, dtype=torch.float32, device=w.device)
    dw.index_add_(0, ids, grad_out.float())
    return out, (dw * scale).to(w.dtype)


# -- one pass ---------------------------------------------------------------------------------

def run(state):
    op = state["op"]
    if not own:
        if op == "sample":
            return _plain_sample(state["logits"], state["uniforms"], state["settings"], state["kept"])
        if op == "kept":
            return _plain_kept(state["logits"], state["labels"], state["kept"], state["temperature"], *state["grads"])
        return _plain_embed(state["ids"], state["weight"], state["scale"], DTYPES[state["out"]], state.get("grad_out"))

    from areal_amd.functional import embed_tokens, gather_kept_logprobs_entropy, sample_tokens

    if op == "sample":
        got = sample_tokens(state["logits"], state["uniforms"], return_kept=state["kept"], **state["settings"])
        out = dict(tokens=got.tokens, logprobs=got.logprobs, full_logprobs=got.full_logprobs)
        if state["kept"]:
            out["kept"] = got.kept
        return out
    if op == "kept":
        lp, ent = gather_kept_logprobs_entropy(state["logits"], state["labels"], state["kept"], state["temperature"])
        (d,) = torch.autograd.grad((lp, ent), state["logits"], state["grads"])
        return lp.detach(), ent.detach(), d
    out = embed_tokens(state["ids"], state["weight"], scale=state["scale"], out_dtype=DTYPES[state["out"]])
    if not state["grad"]:
        return (out,)
    (dw,) = torch.autograd.grad(out, state["weight"], state["grad_out"])
    return out.detach(), dw


# -- the definitions, in 64 bits ---------------------------------------------------------------

def _exact_sample_row(x, u, tau, k, p, min_p):
    """One row: values in order, the cut as a value and a number of ties, the token by bisection."""
    v = x.numel()
    top = x.max()
    if tau <= 0:
        tau, k, full_is_zero = 1.0, 1, True
    else:
        full_is_zero = False
    down = torch.sort(x, descending=True).values
    count = min(k, v) if k > 0 else v
    weights = torch.exp((down[:count] - top) / tau)
    if p < 1:
        mass = torch.cumsum(weights, 0)
        count = min(count, int(torch.searchsorted(mass, p * mass[-1:], right=False)) + 1)
    if min_p > 0:
        count = max(1, min(count, int((weights >= min_p).sum())))
    count = min(count, int((down > -math.inf).sum()))
    cut = down[count - 1]
    above = x > cut
    ties = torch.nonzero(x == cut).view(-1)[: count - int(above.sum())]
    above[ties] = True
    at = torch.nonzero(above).view(-1)
    w = torch.exp((x[at] - top) / tau)
    c = torch.cumsum(w, 0)
    i = min(int(torch.searchsorted(c, u * c[-1:], right=True)), at.numel() - 1)
    exponent = (x[at[i]] - top) / tau
    full = torch.zeros_like(exponent) if full_is_zero else exponent - torch.log(torch.exp((x - top) / tau).sum())
    return int(at[i]), exponent - torch.log(c[-1]), full, above


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "sample":
        x, settings, n = s["logits"], s["settings"], case["rows"]
        def of(name, default):
            value = settings.get(name, default)
            return value.tolist() if torch.is_tensor(value) else [value] * n
        each = list(zip(s["uniforms"].double().tolist(), of("temperature", 1.0), of("top_k", 0), of("top_p", 1.0), of("min_p", 0.0)))
        rows = [_exact_sample_row(x[i].double(), *each[i]) for i in range(n)]
        out = dict(tokens=torch.tensor([r[0] for r in rows]), logprobs=torch.stack([r[1] for r in rows]),
                   full_logprobs=torch.stack([r[2] for r in rows]))
        if case["kept"]:
            out["kept"] = torch.cat([_pack_bits(r[3].unsqueeze(0)) for r in rows])
        return out
    if case["op"] == "kept":
        x, tau = s["logits"].detach(), case["temperature"]
        lps, ents, ds = [], [], []
        for i in range(x.shape[0]):
            word = torch.arange(x.shape[1], device=x.device)
            keep = torch.nonzero((s["kept"][i][word // 32] >> (word % 32).int()) & 1).view(-1)
            z = x[i][keep].double() / tau
            lse = torch.logsumexp(z, 0)
            q = torch.exp(z - lse)
            h = lse - (q * z).sum()
            mine = keep == s["labels"][i]
            glp, gent = s["grads"][0][i].double(), s["grads"][1][i].double()
            d = torch.zeros(x.shape[1], dtype=torch.float64, device=x.device)
            d[keep] = (glp * (mine.double() - q) - gent * q * (z - lse + h)) / tau
            lps.append((z[mine] - lse).squeeze(0))
            ents.append(h)
            ds.append(d.to(x.dtype) if x.shape[0] > 256 else d)  # (many rows in 64 bits are more than is worth holding)
        return torch.stack(lps), torch.stack(ents), torch.stack(ds)
    w, ids = s["weight"].detach(), s["ids"]
    out = w.double().index_select(0, ids) * s["scale"]
    if not case["grad"]:
        return (out,)
    found, which = torch.unique(ids, return_inverse=True)
    sums = torch.zeros(found.numel(), w.shape[1], dtype=torch.float64, device=w.device)
    sums.index_put_((which,), s["grad_out"].double(), accumulate=True)
    dw = torch.zeros(w.shape, dtype=torch.float64, device=w.device)
    dw[found] = sums * s["scale"]
    return out, dw
