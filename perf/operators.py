"""Cases for timing and checking the token operators: embedding lookup and its gradient,
dropout, class log-probabilities and their gradient.

`run` computes a case in plain torch operations, or, where `own` is true, through
rustwood_b200.tokens. Conventions shared by both: an id or target outside the table or the
classes is padding (a zero row, no gradient, log-probability 0); a row of margins that are
all -inf has lse and log-probabilities -inf, log_sum, entropy and gradient 0; equal margins
rank by their index, lowest first. A row's normaliser is kept as its largest margin and the
logarithm of the sum of exponentials relative to it, lse = scale * row_max + log_sum.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZES = {"f32": 4, "bf16": 2, "f16": 2}
ID_DTYPES = {"i32": torch.int32, "i64": torch.int64}

_ctx = None


def _context():
    """The one GPU context that a program keeps for all its calls."""
    global _ctx
    if _ctx is None:
        import rustwood_b200

        _ctx = rustwood_b200.Context(torch.cuda.current_device())
    return _ctx


# ---- cases -----------------------------------------------------------------------------


def listed():
    return [
        # serving: the tokens of one decoding step of a small batch
        {"name": "embed step", "op": "embed", "n": 16, "d": 4096, "vocab": 128000, "dtype": "bf16", "out": "bf16",
         "ids": "i64", "scale": 1.0, "zipf": 1.0, "pad": 0.0},
        # training: the tokens of a batch of 16 sequences of 4096, scaled by sqrt(d)
        {"name": "embed batch", "op": "embed", "n": 65536, "d": 4096, "vocab": 128000, "dtype": "bf16", "out": "bf16",
         "ids": "i64", "scale": 64.0, "zipf": 1.0, "pad": 0.02},
        # a short fine-tuning batch: the dense gradient is mostly zeros
        {"name": "embed grad short", "op": "embed_grad", "n": 512, "d": 768, "vocab": 32000, "dtype": "bf16",
         "out": "f32", "ids": "i64", "scale": 1.0, "zipf": 1.0, "pad": 0.0},
        # the training batch above
        {"name": "embed grad batch", "op": "embed_grad", "n": 65536, "d": 4096, "vocab": 128000, "dtype": "bf16",
         "out": "f32", "ids": "i64", "scale": 64.0, "zipf": 1.0, "pad": 0.02},
        # one categorical column of 50 categories over a million rows, an odd width: long sums
        {"name": "embed grad column", "op": "embed_grad", "n": 1000003, "d": 33, "vocab": 50, "dtype": "f32",
         "out": "f32", "ids": "i32", "scale": 1.0, "zipf": 1.2, "pad": 0.0},
        # a small odd activation
        {"name": "dropout small", "op": "dropout", "rows": 17, "cols": 1001, "dtype": "f32", "p": 0.5},
        # the activations of the training batch
        {"name": "dropout batch", "op": "dropout", "rows": 65536, "cols": 4096, "dtype": "bf16", "p": 0.1},
        # serving: a decoding step, a fifth of the tokens allowed, top 20 reported
        {"name": "logprobs step", "op": "logprobs", "n": 8, "vocab": 128000, "dtype": "bf16", "ids": "i64",
         "scale": 1.25, "top_k": 20, "masked": 0.8, "ignored": 0.0},
        # scoring a batch of given tokens with their entropies and five alternatives
        {"name": "logprobs batch", "op": "logprobs", "n": 4096, "vocab": 128000, "dtype": "bf16", "ids": "i64",
         "scale": 1.0, "top_k": 5, "masked": 0.0, "ignored": 0.05},
        # seven one-vs-rest margins of a million rows
        {"name": "logprobs classes", "op": "logprobs", "n": 1000000, "vocab": 7, "dtype": "f32", "ids": "i32",
         "scale": 1.0, "top_k": 3, "masked": 0.0, "ignored": 0.0},
        # the training loss's gradient, with an entropy term
        {"name": "logprobs grad batch", "op": "logprobs_grad", "n": 4096, "vocab": 128000, "dtype": "bf16",
         "ids": "i64", "scale": 1.0, "entropy": True, "masked": 0.0, "ignored": 0.05},
        # the gradient of the seven margins
        {"name": "logprobs grad classes", "op": "logprobs_grad", "n": 1000000, "vocab": 7, "dtype": "f32",
         "ids": "i32", "scale": 1.0, "entropy": False, "masked": 0.0, "ignored": 0.0},
    ]


def _log(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return int(min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["embed", "embed_grad", "dropout", "logprobs", "logprobs_grad"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    ids = rng.choice(["i64", "i32"])
    if op in ("embed", "embed_grad"):
        d = _log(rng, 8, 8192)
        if rng.random() < 0.6:
            d = max(8, d // 8 * 8)
        vocab = _log(rng, 7, min(262144, (1 << 28) // d))
        n = _log(rng, 1, min(1 << 20, (1 << 28) // d))
        return {"op": op, "n": n, "d": d, "vocab": vocab, "dtype": dtype,
                "out": rng.choice([dtype, "f32"]), "ids": ids,
                "scale": rng.choice([1.0, round(math.sqrt(d), 3)]), "zipf": rng.choice([0.0, 1.0, 1.2]),
                "pad": rng.choice([0.0, 0.1])}
    if op == "dropout":
        cols = _log(rng, 8, 16384)
        if rng.random() < 0.6:
            cols = max(8, cols // 8 * 8)
        return {"op": op, "rows": _log(rng, 1, (1 << 27) // cols), "cols": cols, "dtype": dtype,
                "p": rng.choice([0.05, 0.1, 0.3, 0.5])}
    vocab = _log(rng, 2, 262144)
    if rng.random() < 0.5 and vocab > 64:
        vocab = vocab // 64 * 64
    n = _log(rng, 1, min(1000000, (1 << 28) // vocab))
    case = {"op": op, "n": n, "vocab": vocab, "dtype": dtype, "ids": ids, "scale": rng.choice([1.0, 0.7, 1.25]),
            "masked": rng.choice([0.0, 0.0, 0.5]), "ignored": rng.choice([0.0, 0.1])}
    if op == "logprobs":
        case["top_k"] = min(vocab, rng.choice([0, 1, 5, 20, 32]))
    else:
        case["entropy"] = rng.random() < 0.5
    return case


# ---- inputs ----------------------------------------------------------------------------


def _weights(vocab, zipf):
    return np.arange(1, vocab + 1, dtype=np.float64) ** -zipf


def _ids(gen, n, vocab, zipf, pad, dtype):
    """n ids with Zipf frequencies (0: all alike), the frequent ones anywhere in the table,
    a share of them padding (-1)."""
    cdf = torch.from_numpy(np.cumsum(_weights(vocab, zipf))).cuda()
    u = torch.rand(n, generator=gen, device="cuda", dtype=torch.float64) * cdf[-1]
    rank = torch.searchsorted(cdf, u, right=True).clamp_(max=vocab - 1)
    ids = torch.randperm(vocab, generator=gen, device="cuda")[rank]
    ids[torch.rand(n, generator=gen, device="cuda") < pad] = -1
    return ids.to(ID_DTYPES[dtype])


def _margins(gen, case):
    """Margins with one likely class a row, and the classes asked for: mostly the likely
    ones. With a mask, most classes of a row are -inf, and of one row in 64 all are."""
    n, vocab = case["n"], case["vocab"]
    x = torch.empty(n, vocab, device="cuda", dtype=DTYPES[case["dtype"]])
    x.normal_(0.0, 2.5, generator=gen)
    row = torch.arange(n, device="cuda")
    likely = torch.randint(0, vocab, (n,), generator=gen, device="cuda")
    x[row, likely] += (4.0 + 8.0 * torch.rand(n, generator=gen, device="cuda")).to(x.dtype)
    if case["masked"] > 0:
        out = torch.empty(n, vocab, device="cuda", dtype=torch.uint8).random_(0, 256, generator=gen)
        out = out < int(256 * case["masked"])
        out[row, likely] = False
        out[row % 64 == 5] = True
        x.masked_fill_(out, -math.inf)
    target = torch.where(torch.rand(n, generator=gen, device="cuda") < 0.7, likely,
                         torch.randint(0, vocab, (n,), generator=gen, device="cuda"))
    target[torch.rand(n, generator=gen, device="cuda") < case["ignored"]] = -1
    return x, target.to(ID_DTYPES[case["ids"]])


def _saved(x, scale):
    """What the forward call leaves for its gradient, in 32 bits: row_max, log_sum, entropy."""
    m = x.float().amax(dim=1, keepdim=True)
    dead = m == -math.inf
    d = (x.float() - torch.where(dead, 0.0, m)).mul_(scale)
    e = torch.exp(d)
    s = e.sum(dim=1, keepdim=True)
    t = torch.where(e > 0, e.mul_(d), 0.0).sum(dim=1, keepdim=True)
    log_sum = torch.where(dead, 0.0, torch.log(s))
    h = torch.where(dead, 0.0, log_sum - t / s)
    return m[:, 0].contiguous(), log_sum[:, 0].contiguous(), h[:, 0].contiguous()


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    st = {"case": dict(case)}
    if case["op"] in ("embed", "embed_grad"):
        st["ids"] = _ids(gen, case["n"], case["vocab"], case["zipf"], case["pad"], case["ids"])
        rows = case["vocab"] if case["op"] == "embed" else case["n"]
        std = 0.02 if case["op"] == "embed" else 1e-3
        st["x"] = torch.empty(rows, case["d"], device="cuda", dtype=DTYPES[case["dtype"]]).normal_(0, std, generator=gen)
    elif case["op"] == "dropout":
        st["x"] = torch.empty(case["rows"], case["cols"], device="cuda",
                              dtype=DTYPES[case["dtype"]]).normal_(0, 1, generator=gen)
        st["seed"], st["sequence"] = seed * 0x9E3779B97F4A7C15 % (1 << 64), seed % 1000
    else:
        st["x"], st["target"] = _margins(gen, case)
        if case["op"] == "logprobs_grad":
            st["m"], st["log_sum"], st["h"] = _saved(st["x"], case["scale"])
            n = case["n"]  # a loss summed over the rows, each with its weight
            st["g"] = -(0.5 + torch.rand(n, generator=gen, device="cuda"))
            st["e"] = 0.01 * torch.rand(n, generator=gen, device="cuda") if case["entropy"] else None
    return st


# ---- one pass --------------------------------------------------------------------------


def run(state):
    case, x = state["case"], state["x"]
    op = case["op"]
    if own:
        from rustwood_b200 import tokens

        ctx = _context()
        if op == "embed":
            return tokens.embed(ctx, x, state["ids"], scale=case["scale"], dtype=DTYPES[case["out"]])
        if op == "embed_grad":
            return tokens.embed_grad(ctx, x, state["ids"], case["vocab"], scale=case["scale"], dtype=DTYPES[case["out"]])
        if op == "dropout":
            return tokens.dropout(ctx, x, case["p"], state["seed"], state["sequence"])
        if op == "logprobs":
            r = tokens.logprobs(ctx, x, state["target"], scale=case["scale"], top_k=case["top_k"])
            return {"row_max": r.row_max, "log_sum": r.log_sum, "lse": r.lse, "logp": r.logp, "entropy": r.entropy,
                    "top_logp": r.top_logp, "top_index": r.top_index}
        return tokens.logprobs_grad(ctx, x, state["target"], state["m"], state["log_sum"], state["h"], state["g"],
                                    state["e"], scale=case["scale"])
    if op == "embed":
        return _plain_embed(x, state["ids"], case["scale"], DTYPES[case["out"]])
    if op == "embed_grad":
        return _plain_embed_grad(x, state["ids"], case["vocab"], case["scale"], DTYPES[case["out"]])
    if op == "dropout":
        return _plain_dropout(x, case["p"], state["seed"], state["sequence"])
    if op == "logprobs":
        return _plain_logprobs(x, state["target"], case["scale"], case["top_k"])
    return _plain_logprobs_grad(x, state["target"], state["m"], state["log_sum"], state["h"], state["g"], state["e"],
                                case["scale"])


def _plain_embed(table, ids, scale, dtype):
    ids = ids.long()
    seen = (ids >= 0) & (ids < table.shape[0])
    rows = table[torch.where(seen, ids, 0)].float() * scale
    return torch.where(seen[:, None], rows, 0.0).to(dtype)


def _plain_embed_grad(dout, ids, vocab, scale, dtype):
    # 64 bits: a frequent category's sum has up to a million terms
    ids = ids.long()
    seen = (ids >= 0) & (ids < vocab)
    total = torch.zeros(vocab + 1, dout.shape[1], device=dout.device, dtype=torch.float64)
    total.index_add_(0, torch.where(seen, ids, vocab), dout.double())
    return (total[:vocab] * scale).to(dtype)


def _mul_32(a, b):
    """High and low 32 bits of the product of 32-bit values b (in 64-bit words) and the constant a."""
    low = (a & 0xFFFF) * b
    high = (a >> 16) * b + (low >> 16)
    return high >> 16, ((high & 0xFFFF) << 16) | (low & 0xFFFF)


def _philox(group, sequence, seed):
    """Philox4x32-10 (Salmon, Moraes, Dror and Shaw, 2011): the four words of each counter."""
    c0, c1 = group & 0xFFFFFFFF, group >> 32
    c2 = torch.full_like(c0, sequence & 0xFFFFFFFF)
    c3 = torch.full_like(c0, sequence >> 32)
    k0, k1 = seed & 0xFFFFFFFF, seed >> 32
    for _ in range(10):
        h0, l0 = _mul_32(0xD2511F53, c0)
        h1, l1 = _mul_32(0xCD9E8D57, c2)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return torch.stack([c0, c1, c2, c3], dim=1)


def _plain_dropout(x, p, seed, sequence):
    """Element e is kept where 16 of the generator's bits are at least p: half e % 2 (low
    first) of word (e / 2) % 4 of counter (e / 8, sequence); p counts in 65536ths."""
    n = x.numel()
    limit = round(p * 65536)
    words = _philox(torch.arange((n + 7) // 8, device=x.device), sequence, seed)
    halves = torch.stack([words & 0xFFFF, words >> 16], dim=2).reshape(-1)[:n]
    y = x.float() * (65536.0 / (65536 - limit))
    return torch.where(halves.reshape(x.shape) >= limit, y, 0.0).to(x.dtype)


def _plain_logprobs(x, target, scale, top_k):
    n, vocab = x.shape
    m = x.float().amax(dim=1, keepdim=True)
    dead = m == -math.inf
    d = (x.float() - torch.where(dead, 0.0, m)) * scale
    e = torch.exp(d)
    s = e.sum(dim=1, keepdim=True)
    t = torch.where(e > 0, e * d, 0.0).sum(dim=1, keepdim=True)
    log_sum = torch.where(dead, 0.0, torch.log(s))
    lse = m * scale + log_sum
    entropy = torch.where(dead, 0.0, log_sum - t / s)
    target = target.long()
    seen = (target >= 0) & (target < vocab)
    logp = torch.gather(d, 1, torch.where(seen, target, 0)[:, None]) - log_sum
    logp = torch.where(seen[:, None], logp, 0.0)
    # whole-number keys that rank by value, then by the lower index
    bits = (x.float() + 0.0).view(torch.int32)
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long() * (1 << 32)
    key = torch.topk(order + (vocab - 1 - torch.arange(vocab, device=x.device)), top_k, dim=1).values
    top_index = vocab - 1 - (key & 0xFFFFFFFF)
    top_logp = torch.gather(d, 1, top_index) - log_sum
    return {"row_max": m[:, 0], "log_sum": log_sum[:, 0], "lse": lse[:, 0], "logp": logp[:, 0],
            "entropy": entropy[:, 0], "top_logp": top_logp, "top_index": top_index}


def _plain_logprobs_grad(x, target, row_max, log_sum, h, g, e, scale):
    n, vocab = x.shape
    target = target.long()
    seen = (target >= 0) & (target < vocab)
    dead = (row_max == -math.inf)[:, None]
    g = torch.where(seen, g, 0.0)[:, None]
    logp = (x.float() - torch.where(dead, 0.0, row_max[:, None])) * scale - log_sum[:, None]
    p = torch.where(dead, 0.0, torch.exp(logp))
    grad = -g * p
    if e is not None:
        grad = grad - torch.where(p > 0, e[:, None] * p * (logp + h[:, None]), 0.0)
    row = torch.arange(n, device=x.device)
    at = torch.where(seen, target, 0)
    grad[row, at] += torch.where(dead, 0.0, g)[:, 0]
    return (grad * scale).to(x.dtype)


# ---- what a pass cannot do without -----------------------------------------------------


def _distinct(case):
    """The number of distinct rows that n ids are expected to reach."""
    w = _weights(case["vocab"], case["zipf"])
    q = w / w.sum() * (1.0 - case["pad"])
    return float(np.sum(-np.expm1(case["n"] * np.log1p(-np.minimum(q, 1 - 1e-12)))))


def work(case):
    op = case["op"]
    if op == "embed":
        n, d = case["n"], case["d"]
        rows = _distinct(case)
        return {"bytes": n * int(case["ids"][1:]) // 8 + rows * d * SIZES[case["dtype"]] + n * d * SIZES[case["out"]],
                "flops": n * d}
    if op == "embed_grad":
        n, d = case["n"], case["d"]
        return {"bytes": n * int(case["ids"][1:]) // 8 + n * d * SIZES[case["dtype"]]
                + case["vocab"] * d * SIZES[case["out"]], "flops": n * d + _distinct(case) * d}
    if op == "dropout":
        e = case["rows"] * case["cols"]
        return {"bytes": 2 * e * SIZES[case["dtype"]], "flops": 6 * e}
    e, n, size = case["n"] * case["vocab"], case["n"], SIZES[case["dtype"]]
    ids = n * int(case["ids"][1:]) // 8
    if op == "logprobs":
        return {"bytes": e * size + ids + n * 20 + n * case["top_k"] * 12, "flops": 6 * e}
    return {"bytes": 2 * e * size + ids + n * (20 if case["entropy"] else 12), "flops": (7 if case["entropy"] else 4) * e}


# ---- the definitions in 64 bits --------------------------------------------------------


def exact(case, seed):
    st = prepare(case, seed)
    x = st["x"]
    op = case["op"]
    if op == "embed":
        padded = torch.cat([x, torch.zeros_like(x[:1])])
        ids = st["ids"].long()
        ids = torch.where(ids < 0, x.shape[0], ids)
        return padded.index_select(0, ids).double().mul_(case["scale"])
    if op == "embed_grad":
        # sorted by id; the sum over a run of ids is a difference of two running sums, over
        # blocks of columns
        ids = st["ids"].long()
        ids, perm = torch.sort(ids, stable=True)
        edge = torch.searchsorted(ids, torch.arange(case["vocab"] + 1, device="cuda"))
        out = []
        for cols in torch.split(x, 256, dim=1):
            run_sum = torch.zeros(case["n"] + 1, cols.shape[1], device="cuda", dtype=torch.float64)
            torch.cumsum(cols[perm].double(), dim=0, out=run_sum[1:])
            out.append((run_sum[edge[1:]] - run_sum[edge[:-1]]) * case["scale"])
        return torch.cat(out, dim=1)
    if op == "dropout":
        n = x.numel()
        limit = round(case["p"] * 65536)
        words = _exact_words((n + 7) // 8, st["sequence"], st["seed"])
        keep = torch.cat([torch.stack([w % 65536, w // 65536], 1) for w in words], 1).reshape(-1)[:n] >= limit
        return x.double() * keep.reshape(x.shape) / (1.0 - limit / 65536)
    z = x.double().mul_(case["scale"])
    lse = torch.logsumexp(z, dim=1)
    lp = z - lse[:, None]
    lp = torch.where(torch.isnan(lp), -math.inf, lp)
    if op == "logprobs":
        ranked = torch.argsort(x.double(), dim=1, descending=True, stable=True)[:, :case["top_k"]] \
            if x.numel() < (1 << 27) else _exact_top(x, case["top_k"])
        top = torch.gather(lp, 1, ranked)
        t = st["target"].long()
        logp = torch.where(t < 0, 0.0, lp.gather(1, t.clamp(min=0)[:, None])[:, 0])
        h = torch.special.entr(lp.exp_()).sum(dim=1)
        m = x.double().amax(dim=1)
        log_sum = torch.where(torch.isinf(m), 0.0, lse - case["scale"] * m)
        return {"row_max": m, "log_sum": log_sum, "lse": lse, "logp": logp, "entropy": h, "top_logp": top, "top_index": None}
    # the gradient of sum(g logp + e H) as p times the differences from its mean, with the
    # definition's own lse and entropy
    p = lp.exp()
    t = st["target"].long()
    dlogp = torch.zeros_like(p)
    dlogp.scatter_(1, t.clamp(min=0)[:, None], torch.where(t < 0, 0.0, st["g"].double())[:, None])
    if st["e"] is not None:
        dlogp -= st["e"].double()[:, None] * torch.where(p > 0, p * (lp + 1.0), 0.0)
    dlogp = torch.where(torch.isinf(lse)[:, None], 0.0, dlogp)
    return (dlogp - p * dlogp.sum(dim=1, keepdim=True)) * case["scale"]


def _exact_top(x, k):
    """The first k of each row by repeated choice of the first largest value."""
    left, out = x.clone(), []
    col = torch.arange(x.shape[1], device=x.device)
    for _ in range(k):
        best = left.amax(dim=1, keepdim=True)
        first = torch.where(left == best, col, x.shape[1]).amin(dim=1, keepdim=True)
        out.append(first)
        left.scatter_(1, first, float("nan"))
        left = torch.where(torch.isnan(left), -math.inf, left)
    return torch.cat(out, dim=1)


def _exact_words(count, sequence, seed):
    """The generator's words with products in 64-bit floating point: 32 by 16 bits at a time
    stays below 2^53."""
    def product(a, w):
        lo = (w * float(a % 65536))
        hi = (w * float(a // 65536)) + torch.floor(lo / 65536)
        return torch.floor(hi / 65536).long(), (torch.remainder(hi, 65536) * 65536 + torch.remainder(lo, 65536)).long()

    w = [torch.arange(count, device="cuda"), torch.zeros(count, dtype=torch.int64, device="cuda")]
    w += [torch.full((count,), sequence % (1 << 32), device="cuda"), torch.full((count,), sequence // (1 << 32), device="cuda")]
    for r in range(10):
        key = [(seed + r * 0x9E3779B9) % (1 << 32), (seed // (1 << 32) + r * 0xBB67AE85) % (1 << 32)]
        a, b = product(0xD2511F53, w[0].double()), product(0xCD9E8D57, w[2].double())
        w = [b[0] ^ w[1] ^ key[0], b[1], a[0] ^ w[3] ^ key[1], a[1]]
    return w
