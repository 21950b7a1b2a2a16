"""The token operators on the GPU against plain implementations in 64 bits.

Tolerances count roundings, each at most half a step (2^-24 relative for f32, 2^-8 bf16,
2^-11 f16). A sum of m terms in f32 is off by at most m * 2^-24 times the sum of the terms'
magnitudes; exponentials and logarithms of d carry d's own rounding (|d| * 2^-23 for the
difference and its scaling) and a few units of the function (2^-21 together).
"""
import math

import numpy as np
import pytest
import torch

from rustwood_b200 import _native as N

pytestmark = pytest.mark.gpu
if torch.cuda.is_available():
    from rustwood_b200 import tokens

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [F32, BF16, F16]
U = 2.0 ** -24
INF, NAN = math.inf, math.nan


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rand(seed, *shape, dtype=F32, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.empty(shape, device="cuda", dtype=dtype).normal_(0, std, generator=g)


def rand_ids(seed, n, vocab, skew=1.0, dtype=torch.int64, pad=0.1):
    rng = np.random.default_rng(seed)
    q = np.arange(1, vocab + 1) ** -float(skew)
    ids = rng.permutation(vocab)[rng.choice(vocab, size=n, p=q / q.sum())]
    ids[rng.random(n) < pad] = rng.choice([-1, -100, vocab, vocab + 7])
    return torch.from_numpy(ids).to("cuda", dtype)


def strided(t, extra=3):
    """The same values with rows further apart and a base that is not 16-byte aligned."""
    rows, cols = t.shape
    buf = torch.full((rows * (cols + extra) + 1,), NAN, device="cuda", dtype=t.dtype)
    v = buf[1:].as_strided((rows, cols), (cols + extra, 1))
    v.copy_(t)
    return v


# ---- embedding ---------------------------------------------------------------------------


@pytest.mark.parametrize("n,d,vocab", [(1, 1, 1), (3, 8, 5), (17, 33, 100), (1000, 64, 7),
                                       (257, 500, 999), (64, 4096, 300), (5, 8200, 40), (0, 8, 5)])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_embed(ctx, n, d, vocab, dtype):
    table = rand(1, vocab, d, dtype=dtype)
    for id_type, scale, out in ((torch.int64, 1.0, None), (torch.int32, 0.37, F32), (torch.int64, -3.0, BF16)):
        ids = rand_ids(n + d, n, vocab, dtype=id_type)
        safe = ids.long().clamp(0, vocab - 1)
        seen = (ids >= 0) & (ids < vocab)
        want = torch.where(seen[:, None], table[safe].float() * scale, 0.0).to(out or dtype)
        for t in (table, strided(table)):
            got = tokens.embed(ctx, t, ids, scale=scale, dtype=out)
            assert torch.equal(got, want)


def test_embed_shapes_and_outputs(ctx):
    table = rand(2, 50, 24, dtype=BF16)
    ids = rand_ids(3, 30, 50).reshape(2, 5, 3)
    got = tokens.embed(ctx, table, ids)
    assert got.shape == (2, 5, 3, 24) and got.dtype == BF16
    flat = got.reshape(30, 24)
    assert torch.equal(tokens.embed(ctx, table, ids.transpose(0, 2)), got.transpose(0, 2))
    # into the middle of a wider buffer, whose other columns stay
    buf = torch.full((30, 40), 7.0, device="cuda", dtype=BF16)
    tokens.embed(ctx, table, ids.reshape(30), out=buf[:, 8:32])
    assert torch.equal(buf[:, 8:32], flat)
    assert (buf[:, :8] == 7).all() and (buf[:, 32:] == 7).all()
    # a transposed table is copied, not misread
    assert torch.equal(tokens.embed(ctx, table.t().contiguous().t(), ids), got)
    none = tokens.embed(ctx, table[:0], ids)
    assert (none == 0).all()
    assert tokens.embed(ctx, table[:, :0], ids).shape == (2, 5, 3, 0)
    with pytest.raises(ValueError):
        tokens.embed(ctx, table, ids, out=torch.empty(30, 24, device="cuda", dtype=BF16))
    with pytest.raises(TypeError):
        tokens.embed(ctx, table.double(), ids)
    with pytest.raises(TypeError):
        tokens.embed(ctx, table, ids.float())


def grad_reference(grad, ids, vocab, scale):
    """(sum, sum of magnitudes, terms) per row in 64 bits."""
    seen = (ids >= 0) & (ids < vocab)
    at = torch.where(seen, ids.long(), vocab)
    total = torch.zeros(vocab + 1, grad.shape[1], device="cuda", dtype=torch.float64)
    size, count = torch.zeros_like(total), torch.zeros(vocab + 1, device="cuda", dtype=torch.float64)
    total.index_add_(0, at, grad.double() * scale)
    size.index_add_(0, at, grad.double().abs() * abs(scale))
    count.index_add_(0, at, torch.ones(len(at), device="cuda", dtype=torch.float64))
    return total[:vocab], size[:vocab], count[:vocab]


def check_grad(got, grad, ids, vocab, scale, start=None):
    want, size, count = grad_reference(grad, ids, vocab, scale)
    if start is not None:
        want, size = want + start.double(), size + start.double().abs()
    # count additions, the scaling, the addition of the old value; then the output's rounding
    tol = (count[:, None] + 3) * U * size + half_step(got.dtype) * want.abs() + 1e-30
    if got.dtype == F16:
        tol = tol + 2.0 ** -25  # half of its smallest step
    off = (got.double() - want).abs()
    assert (off <= tol).all(), float((off - tol).max())
    assert (got[count == 0] == (0 if start is None else start[count == 0])).all()


GRAD_SIZES = [(1, 1, 1), (2, 3, 2), (100, 8, 1), (511, 33, 50), (513, 64, 511), (4097, 16, 512),
              (5000, 40, 70000), (9000, 24, 300000), (20011, 5, 3), (70001, 8, 1000),
              (300, 2056, 40), (37, 8200, 9), (1000, 512, 2)]


@pytest.mark.parametrize("n,d,vocab", GRAD_SIZES)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_embed_grad(ctx, n, d, vocab, dtype):
    for skew, id_type, scale, out in ((1.2, torch.int64, 1.0, F32), (0.0, torch.int32, -0.5, dtype)):
        ids = rand_ids(n + d, n, vocab, skew, id_type)
        grad = rand(n, n, d, dtype=dtype)
        got = tokens.embed_grad(ctx, grad, ids, vocab, scale=scale, dtype=out)
        check_grad(got, grad, ids, vocab, scale)
        again = tokens.embed_grad(ctx, strided(grad), ids, vocab, scale=scale, dtype=out)
        check_grad(again, grad, ids, vocab, scale)
        assert torch.equal(tokens.embed_grad(ctx, grad, ids, vocab, scale=scale, dtype=out), got)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_embed_grad_accumulates(ctx, dtype):
    for n, d, vocab in ((3000, 40, 900), (20000, 33, 7), (5, 64, 30000)):
        ids = rand_ids(n, n, vocab)
        grad = rand(n, n, d, dtype=dtype)
        buf = rand(5, vocab, d + 8, dtype=dtype)
        start = buf.clone()
        out = buf[:, :d]
        assert tokens.embed_grad(ctx, grad, ids, vocab, scale=2.0, out=out, accumulate=True) is out
        check_grad(out, grad, ids, vocab, 2.0, start[:, :d])
        assert torch.equal(buf[:, d:], start[:, d:])


def test_embed_grad_of_no_ids(ctx):
    out = rand(1, 10, 8)
    kept = out.clone()
    none = torch.empty(0, dtype=torch.int64, device="cuda")
    tokens.embed_grad(ctx, rand(2, 0, 8), none, 10, out=out, accumulate=True)
    assert torch.equal(out, kept)
    assert (tokens.embed_grad(ctx, rand(2, 0, 8), none, 10, out=out) == 0).all()
    pad = torch.full((500,), -1, device="cuda")
    assert (tokens.embed_grad(ctx, rand(2, 500, 8), pad, 10) == 0).all()
    assert tokens.embed_grad(ctx, rand(2, 500, 8), pad, 0).shape == (0, 8)
    with pytest.raises(ValueError):
        tokens.embed_grad(ctx, rand(2, 500, 8), pad, 10, accumulate=True)
    with pytest.raises(ValueError):
        tokens.embed_grad(ctx, rand(2, 499, 8), pad, 10)


def test_embed_grad_keeps_nan_to_its_row(ctx):
    ids = torch.arange(2000, device="cuda") % 5
    grad = rand(1, 2000, 16)
    grad[3, 4] = NAN     # id 3
    grad[1001, 0] = INF  # id 1
    got = tokens.embed_grad(ctx, grad, ids, 8)
    bad = ~torch.isfinite(got)
    assert bad[3, 4] and bad[1, 0] and int(bad.sum()) == 2
    assert (got[5:] == 0).all()


def test_embed_and_its_gradient_are_adjoint(ctx):
    """<embed(T), G> = <T, embed_grad(G)>, and a difference of embed along G's direction."""
    ids = rand_ids(4, 777, 60)
    table, grad = rand(1, 60, 48), rand(2, 777, 48)
    left = (tokens.embed(ctx, table, ids, scale=1.5).double() * grad.double()).sum()
    dt = tokens.embed_grad(ctx, grad, ids, 60, scale=1.5)
    right = (table.double() * dt.double()).sum()
    size = (dt.double().abs() * table.double().abs()).sum()
    assert abs(left - right) <= 400 * U * size + 777 * 48 * U
    step = 0.125
    up = (tokens.embed(ctx, table + step * dt, ids, scale=1.5).double() * grad.double()).sum()
    want = (dt.double() ** 2).sum() * step
    # table + step * dt is rounded once per element, and every embedded value once
    tol = (2 * U * (table.double().abs() + step * dt.double().abs()) * dt.double().abs()).sum() * 4 \
        + 1000 * U * want + 4 * U * (grad.double().abs() * 20).sum()
    assert abs((up - left) - want) <= tol


def test_lookup_and_its_gradient_past_32_bit_offsets(ctx):
    """2^31 elements lie before the last rows of the output, and of the gradient that is summed."""
    n, d = 530000, 4096
    table = rand(1, 20, d, dtype=BF16)
    ids = torch.arange(n, device="cuda") % 20
    x = tokens.embed(ctx, table, ids)
    assert torch.equal(x[-20:], table[ids[-20:]]) and torch.equal(x[:20], table)
    x.zero_()
    x[-40:] = rand(2, 40, d, dtype=BF16)
    got = tokens.embed_grad(ctx, x, ids, 25)
    check_grad(got, x[-40:], ids[-40:], 25, 1.0)


# ---- dropout -----------------------------------------------------------------------------


def philox_keep(n, p, seed, sequence, first=0):
    """Which of n elements from `first` (a multiple of 8) on are kept, in numpy 64-bit integers
    (Philox4x32-10)."""
    m32 = np.uint64(0xFFFFFFFF)
    g = np.arange((n + 7) // 8, dtype=np.uint64) + np.uint64(first // 8)
    c = [g & m32, g >> np.uint64(32), np.full_like(g, sequence & 0xFFFFFFFF), np.full_like(g, sequence >> 32)]
    k0, k1 = seed & 0xFFFFFFFF, seed >> 32
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k0), b & m32,
             (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k1), a & m32]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    halves = np.stack([h for w in c for h in (w & np.uint64(0xFFFF), w >> np.uint64(16))], 1).reshape(-1)
    return halves[:n] >= np.uint64(round(p * 65536))


def test_philox_known_answers():
    """The published test vectors of Philox4x32-10 (zero and all-ones counter and key)."""
    def words(counter, key):
        c, (k0, k1) = list(counter), key
        for _ in range(10):
            a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
            c = [(b >> 32) ^ c[1] ^ k0, b & 0xFFFFFFFF, (a >> 32) ^ c[3] ^ k1, a & 0xFFFFFFFF]
            k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
        return c
    ones = 0xFFFFFFFF
    assert words([0] * 4, (0, 0)) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert words([ones] * 4, (ones, ones)) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    keep = philox_keep(8, 0x8000 / 65536, 0, 0)
    flat = [h for w in words([0] * 4, (0, 0)) for h in (w & 0xFFFF, w >> 16)]
    assert keep.tolist() == [h >= 0x8000 for h in flat]


@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 7), (3, 8), (17, 1001), (300, 64), (1, 100003), (5, 4096)])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_dropout(ctx, rows, cols, dtype):
    x = rand(rows, rows, cols, dtype=dtype)
    for p, seed, seq in ((0.1, 1, 0), (0.5, (1 << 64) - 3, (1 << 63) + 5), (0.999, 1 << 40, 77)):
        keep = torch.from_numpy(philox_keep(rows * cols, p, seed, seq)).cuda().reshape(rows, cols)
        scale = 65536.0 / (65536 - round(p * 65536))
        want = torch.where(keep, x.float() * scale, 0.0).to(dtype)
        assert torch.equal(tokens.dropout(ctx, x, p, seed, seq), want)
        assert torch.equal(tokens.dropout(ctx, strided(x), p, seed, seq), want)
        out = strided(torch.zeros_like(x))
        tokens.dropout(ctx, x, p, seed, seq, out=out)
        assert torch.equal(out, want)
        y = x.clone()
        assert tokens.dropout(ctx, y, p, seed, seq, out=y) is y and torch.equal(y, want)
        offset = torch.cat([x.reshape(-1)[:1], x.reshape(-1)])[1:]  # one element off alignment
        assert torch.equal(tokens.dropout(ctx, offset, p, seed, seq), want.reshape(-1))


@pytest.mark.parametrize("extra", [0, 3])
def test_dropout_past_32_bit_offsets(ctx, extra):
    """Elements around and beyond 2^31, contiguous and with rows further apart."""
    rows, cols = 530000, 4096
    buf = torch.ones(rows, cols + extra, device="cuda", dtype=BF16)
    x = buf[:, :cols]
    tokens.dropout(ctx, x, 0.25, 5, 6, out=x)
    for row in (0, 524288, rows - 2):
        keep = philox_keep(2 * cols, 0.25, 5, 6, first=row * cols)
        want = torch.from_numpy(keep).cuda().reshape(2, cols) * torch.tensor(4 / 3, device="cuda")
        assert torch.equal(x[row:row + 2], want.to(BF16))
    assert (buf[:, cols:] == 1).all()


def test_dropout_ends_of_p(ctx):
    x = rand(1, 100, 33)
    x[5] = NAN
    x[6] = INF
    assert torch.equal(tokens.dropout(ctx, x, 1.0, 3), torch.zeros_like(x))
    got = tokens.dropout(ctx, x, 0.0, 3)
    assert torch.equal(got.nan_to_num(9.0), x.nan_to_num(9.0))
    y = tokens.dropout(ctx, x, 0.25, 3, 4)
    keep = torch.from_numpy(philox_keep(3300, 0.25, 3, 4)).cuda().reshape(100, 33)
    assert (y[5][~keep[5]] == 0).all() and y[5][keep[5]].isnan().all()
    assert (y[6][~keep[6]] == 0).all() and (y[6][keep[6]] == INF).all()
    assert tokens.dropout(ctx, x[:0], 0.5, 3).shape == (0, 33)
    # the share kept: 40,000 draws of variance p (1 - p), six deviations
    z = tokens.dropout(ctx, torch.ones(40000, device="cuda"), 0.3, 9)
    assert abs(float((z == 0).float().mean()) - 0.3) < 6 * math.sqrt(0.21 / 40000)


# ---- log-probabilities ---------------------------------------------------------------------


def logprob_reference(x, targets, scale, k):
    """In 64 bits, rows without NaN or +inf."""
    x = x.double()
    m = x.amax(1) if x.shape[1] else torch.full((x.shape[0],), -INF, device="cuda", dtype=torch.float64)
    dead = m == -INF
    d = (x - torch.where(dead, 0.0, m)[:, None]) * scale
    e = d.exp()
    s = e.sum(1)
    log_sum = torch.where(dead, 0.0, s.log())
    ent = torch.where(dead, 0.0, log_sum - torch.where(e > 0, e * d, 0.0).sum(1) / s)
    lp = d - log_sum[:, None]
    seen = (targets >= 0) & (targets < x.shape[1])
    at = torch.where(seen, targets.long(), 0)
    logp = torch.where(seen, lp.gather(1, at[:, None])[:, 0], 0.0) if x.shape[1] else torch.zeros_like(m)
    order = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :k]
    return m, log_sum, scale * m + log_sum, logp, ent, lp.gather(1, order), order, d


def check_logprobs(got, x, targets, scale, k):
    m, log_sum, lse, logp, ent, top, order, d = logprob_reference(x, targets, scale, k)
    v = x.shape[1]
    # the sum: at least 256 running sums when there are many classes; every term's own error
    deep = (v if v <= 1024 else v / 256 + 40) * U
    tol_s = deep + math.log(max(v, 2)) * 2 * U + 8 * U

    def near(a, b, tol):
        a = a.double()
        same = a == b  # infinities
        assert (same | ((a - b).abs() <= tol)).all(), float(torch.where(same, 0.0, (a - b).abs() - tol).max())

    assert torch.equal(got.row_max.double(), m)
    near(got.log_sum, log_sum, tol_s + U * log_sum.abs())
    near(got.lse, lse, tol_s + 2 * U * (lse.abs() + (scale * m).abs()))
    assert torch.equal(got.top_index, order)

    def logp_tol(b):
        size = torch.where(torch.isfinite(b), b.abs(), 0.0)
        return tol_s + 2 * U * (size + math.log(max(v, 2))) + U * size

    near(got.top_logp, top, logp_tol(top))
    if got.logp is not None:
        near(got.logp, logp, logp_tol(logp))
    # the weighted sum of d: terms off by their own rounding (|d| counts up to 30, where e^d
    # ends to matter) and the summation
    near(got.entropy, ent, tol_s + ent.abs() * (2 * tol_s + 60 * U) + 4 * U * ent.abs())


LOGPROB_SIZES = [(1, 1), (3, 2), (50, 7), (33, 31), (65, 32), (40, 100), (9, 500), (20, 1024),
                 (5, 1025), (7, 4099), (3, 50001), (1, 128000), (2, 262144), (300, 2048), (0, 5)]


def margins(seed, n, v, dtype, std=3.0):
    x = rand(seed, n, v, dtype=dtype, std=std)
    rng = np.random.default_rng(seed)
    t = rng.integers(0, v, n)
    t[rng.random(n) < 0.1] = rng.choice([-1, -100, v, v + 3])
    return x, torch.from_numpy(t).cuda()


@pytest.mark.parametrize("n,v", LOGPROB_SIZES)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_logprobs(ctx, n, v, dtype):
    x, t = margins(n + v, n, v, dtype)
    for k, scale, kind in ((min(v, 5), 1.0, torch.int64), (min(v, 32), 0.3, torch.int32), (0, 2.5, torch.int64)):
        got = tokens.logprobs(ctx, x, t.to(kind), scale=scale, top_k=k)
        check_logprobs(got, x, t, scale, k)
        other = tokens.logprobs(ctx, strided(x), t.to(kind), scale=scale, top_k=k)
        check_logprobs(other, x, t, scale, k)
        again = tokens.logprobs(ctx, x, t.to(kind), scale=scale, top_k=k)
        assert all(torch.equal(p, q) for p, q in zip(got, again))
    got = tokens.logprobs(ctx, x, top_k=min(v, 1))
    assert got.logp is None
    check_logprobs(got, x, t, 1.0, min(v, 1))


@pytest.mark.parametrize("v", [2, 7, 20, 40, 300, 1024, 3000, 40000, 140000])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_logprobs_masks_and_ties(ctx, v, dtype):
    """Rows with nothing left, one class left, few left, the type's lowest value as the mask,
    all equal, rising and falling values, many ties around the last place."""
    low = torch.finfo(dtype).min
    x, t = margins(v, 14, v, dtype)
    x[0] = -INF
    x[1] = -INF
    x[1, v - 1] = 2.0
    x[2] = -INF
    x[2, ::max(1, v // 3)] = 1.0
    x[3] = low
    x[4] = low
    x[4, v // 2] = -5.0
    x[5] = 0.25
    x[6] = torch.linspace(-8, 8, v, device="cuda").to(dtype)
    x[7] = x[6].flip(0)
    x[8] = torch.arange(v, device="cuda").remainder(3).to(dtype)
    x[9] = 0.0
    x[9, 1::2] = -0.0
    x[10] = torch.where(torch.arange(v, device="cuda") < v // 2, 1.0, 4.0).to(dtype)
    x[11, 0] = low
    x[11, v - 1] = -INF
    x[12, v // 2:] = -INF
    x[13, : v - 1] = -INF
    t[:7] = torch.tensor([0, v - 1, 1, 0, v // 2, 1, 0], device="cuda")
    for k in {0, 1, min(v, 3), min(v, 20), min(v, 32)}:
        for scale in (1.0, 0.5):
            check_logprobs(tokens.logprobs(ctx, x, t, scale=scale, top_k=k), x, t, scale, k)
            check_logprobs(tokens.logprobs(ctx, strided(x), t, scale=scale, top_k=k), x, t, scale, k)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_logprobs_largest_margins_side_by_side(ctx, dtype):
    """The largest margins lie 8 (4) at a time every 256 vectors, all in few threads' shares."""
    v = 140000
    x, t = margins(1, 3, v, dtype)
    per = 16 // x.element_size()
    at = torch.arange(v, device="cuda")
    share = (at // per) % 256
    for row, threads in ((0, 4), (1, 9), (2, 31)):
        x[row] += torch.where(share < threads, 30.0, 0.0).to(dtype)
    for k in (1, 5, 32):
        check_logprobs(tokens.logprobs(ctx, x, t, top_k=k), x, t, 1.0, k)
        one = tokens.logprobs(ctx, x[:1].repeat(600, 1), t[:1].repeat(600), top_k=k)  # rows not split
        assert torch.equal(one.top_index, tokens.logprobs(ctx, x[:1], t[:1], top_k=k).top_index.expand(600, k))


@pytest.mark.parametrize("v", [7, 100, 900, 1500, 30000])
def test_logprobs_far_margins_and_scales(ctx, v):
    """Margins near the ends of f32's range, a shared offset, and scales far from 1."""
    x, t = margins(v, 5, v, F32)
    x[1] *= 5e37
    x[2] += 4096.0
    x[3] = -3e38
    x[3, v // 2] = -2.9e38
    x[4] *= 1e-12
    x, t = torch.cat([x, x[:1] * 2e37]), torch.cat([t, t[:1]])
    # beyond 900 classes some margins of row 1 are above 3.4e38 / 5e37 and so +inf
    over = x.isposinf().any(1)
    for scale in (1.0, 1e-19, 1e-7, 1e7, 1e19):
        r = tokens.logprobs(ctx, x, t, scale=scale, top_k=2)
        assert r.log_sum[over].isnan().all() and r.entropy[over].isnan().all()
        r = type(r)(*(f[~over] for f in r))
        check_far_margins(ctx, x[~over], t[~over], scale, v, r)


def check_far_margins(ctx, x, t, scale, v, r):
    m, log_sum, _, logp, ent, _, order, _ = logprob_reference(x, t, scale, 2)
    # d = scale (x - m) is off by |d| 2^-23: the sum's terms by |d| e^d 2^-23, and |d| e^d
    # is below 0.37, so the sum of at most v of them is off by v * 0.37 * 2^-23 at most
    tol = (v * 0.74 + 64 + v / 128) * U
    assert torch.equal(r.top_index, order)
    assert ((r.log_sum.double() - log_sum).abs() <= tol + U * log_sum).all()
    big = logp.abs() * 4 * U + tol
    f32_range = logp.abs() < 3e38  # beyond it, -inf
    assert ((r.logp.double() - logp).abs() <= big)[f32_range].all()
    assert (r.logp[~f32_range] == -INF).all()
    # the terms d e^d: their size times their own relative error, |d| 2^-22 and less
    assert ((r.entropy.double() - ent).abs() <= 4 * tol + 8 * U * ent).all()
    g, e = -torch.ones(len(x), device="cuda"), torch.full((len(x),), 0.5, device="cuda")
    got = tokens.logprobs_grad(ctx, x, t, r.row_max, r.log_sum, r.entropy, g, e, scale=scale)
    check_logprobs_grad(got, x, t, r.row_max, r.log_sum, r.entropy, g, e, scale)


@pytest.mark.parametrize("v", [5, 30, 700, 5000, 140000])
def test_logprobs_of_nan_and_infinity(ctx, v):
    x, t = margins(v, 5, v, F32)
    t[:] = 0
    x[1, v // 2] = NAN
    x[2, v - 1] = INF
    x[3, 1] = -NAN
    x[3, v - 2] = INF
    k = min(v, 4)
    got = tokens.logprobs(ctx, x, t, top_k=k)
    fine = torch.tensor([0, 4], device="cuda")
    check_logprobs(type(got)(*(f[fine] for f in got)), x[fine], t[fine], 1.0, k)
    for r in (1, 2, 3):
        for f in (got.log_sum, got.lse, got.logp, got.entropy):
            assert f[r].isnan()
        assert got.top_logp[r].isnan().all()
    assert got.row_max[1].isnan() and got.row_max[2] == INF and got.row_max[3].isnan()
    key = x.nan_to_num(nan=1e30, posinf=1e29)  # NaN ranks above +inf
    order = torch.sort(key, dim=1, descending=True, stable=True).indices[:, :k]
    assert torch.equal(got.top_index, order)


def test_logprobs_shapes(ctx):
    x, t = margins(3, 24, 60, BF16)
    flat = tokens.logprobs(ctx, x, t, top_k=4)
    got = tokens.logprobs(ctx, x.reshape(2, 3, 4, 60), t.reshape(2, 3, 4), top_k=4)
    assert got.logp.shape == (2, 3, 4) and got.top_index.shape == (2, 3, 4, 4)
    assert all(torch.equal(a.reshape(b.shape), b) for a, b in zip(got, flat))
    # one row shown many times, and a single row without a batch
    many = tokens.logprobs(ctx, x[:1].expand(5, 60), t[:1].expand(5), top_k=4)
    assert torch.equal(many.lse, flat.lse[:1].expand(5))
    one = tokens.logprobs(ctx, x[0], t[0], top_k=4)
    assert one.lse.shape == () and torch.equal(one.top_index, flat.top_index[0])
    none = tokens.logprobs(ctx, x[:, :0], t)
    assert (none.lse == -INF).all() and (none.logp == 0).all() and (none.entropy == 0).all()
    with pytest.raises(ValueError):
        tokens.logprobs(ctx, x, t[:-1])
    with pytest.raises(N.RwError):
        tokens.logprobs(ctx, x, t, top_k=33)
    with pytest.raises(N.RwError):
        tokens.logprobs(ctx, x[:, :3], t, top_k=4)
    with pytest.raises(N.RwError):
        tokens.logprobs(ctx, x, t, scale=0.0)


def test_logprobs_past_32_bit_offsets(ctx):
    """2^31 elements lie before the last row."""
    n, v = 16500, 131072
    x = torch.zeros(n, v, device="cuda", dtype=BF16)
    x[n - 1] = rand(1, v, dtype=BF16)
    x[n - 2, v - 1] = 9.0
    t = torch.full((n,), v - 1, device="cuda")
    got = tokens.logprobs(ctx, x, t, top_k=3)
    tail = type(got)(*(f[-3:] for f in got))
    check_logprobs(tail, x[-3:], t[-3:], 1.0, 3)
    assert (got.lse[:-2] == got.lse[0]).all()
    g = -torch.ones(n, device="cuda")
    tokens.logprobs_grad(ctx, x, t, got.row_max, got.log_sum, None, g, out=x)
    assert (x[: n - 2] == x[0]).all() and float(x[n - 1].float().sum().abs()) < 0.05


# ---- its gradient ------------------------------------------------------------------------------


def grad_of_logprobs(x, t, m, log_sum, h, g, e, scale):
    x, m, log_sum, h, g, e = (v.double() for v in (x, m, log_sum, h, g, e))
    v = x.shape[1]
    dead = (m == -INF)[:, None]
    lp = (x - torch.where(dead[:, 0], 0.0, m)[:, None]) * scale - log_sum[:, None]
    p = torch.where(dead, 0.0, lp.exp())
    seen = ((t >= 0) & (t < v)) & ~dead[:, 0]
    g = torch.where(seen, g, 0.0)
    hit = torch.zeros_like(x)
    if v:
        hit.scatter_(1, torch.where(seen, t.long(), 0)[:, None], torch.where(seen, 1.0, 0.0)[:, None].double())
    lph = torch.where(p > 0, lp + h[:, None], 0.0)
    want = scale * (g[:, None] * (hit - p) - e[:, None] * p * lph)
    # p is off by its exponent's rounding and the exponential's; the products by a few units
    size = torch.where(p > 0, lp.abs(), 0.0)
    rel = (2 * size + 3 * log_sum.abs()[:, None] + 16) * U
    tol = scale * (p * (g.abs()[:, None] + e.abs()[:, None] * (lph.abs() + size + h[:, None] + 1)) * rel
                   + 4 * U * g.abs()[:, None] * hit)
    return want, tol


def check_logprobs_grad(got, *args):
    want, tol = grad_of_logprobs(*args)
    tol = tol + half_step(got.dtype) * (want.abs() + tol) + 1e-37
    if got.dtype == F16:
        tol = tol + 2.0 ** -25
    off = (got.double() - want).abs()
    assert (off <= tol).all(), float((off - tol).max())


@pytest.mark.parametrize("n,v", LOGPROB_SIZES)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_logprobs_grad(ctx, n, v, dtype):
    x, t = margins(n + 2 * v, n, v, dtype)
    if n > 2:
        x[1] = -INF
        x[2, ::2] = -INF
    for scale, kind in ((1.0, torch.int64), (0.6, torch.int32)):
        m, log_sum, _, _, h = (f.float() for f in logprob_reference(x, t, scale, 0)[:5])
        g, e = rand(1, n), rand(2, n)
        zero = torch.zeros_like(g)
        tk = t.to(kind)
        got = tokens.logprobs_grad(ctx, x, tk, m, log_sum, h, g, e, scale=scale)
        check_logprobs_grad(got, x, t, m, log_sum, h, g, e, scale)
        got = tokens.logprobs_grad(ctx, strided(x), tk, m, log_sum, None, g, scale=scale)
        check_logprobs_grad(got, x, t, m, log_sum, h, g, zero, scale)
        got = tokens.logprobs_grad(ctx, x, None, m, log_sum, h, None, e, scale=scale)
        check_logprobs_grad(got, x, t, m, log_sum, h, zero, e, scale)
        out = strided(torch.zeros_like(x))
        tokens.logprobs_grad(ctx, x, tk, m, log_sum, h, g, e, scale=scale, out=out)
        check_logprobs_grad(out, x, t, m, log_sum, h, g, e, scale)
        y = x.clone()
        tokens.logprobs_grad(ctx, y, tk, m, log_sum, h, g, e, scale=scale, out=y)
        check_logprobs_grad(y, x, t, m, log_sum, h, g, e, scale)


@pytest.mark.parametrize("v", [4, 50, 2000, 9001])
def test_logprobs_grad_masks(ctx, v):
    for dtype in TYPES:
        x, t = margins(v, 6, v, dtype)
        x[0] = -INF
        x[1] = torch.finfo(dtype).min       # nothing left, by the lowest value: uniform
        x[2, 1:] = torch.finfo(dtype).min
        x[3, : v // 2] = -INF
        t = torch.tensor([0, 1, 0, 0, -1, v], device="cuda")  # t[3] is a masked class
        r = tokens.logprobs(ctx, x, t)
        g, e = -torch.ones(6, device="cuda"), torch.full((6,), 0.1, device="cuda")
        got = tokens.logprobs_grad(ctx, x, t, r.row_max, r.log_sum, r.entropy, g, e)
        check_logprobs_grad(got, x, t, r.row_max, r.log_sum, r.entropy, g, e, 1.0)
        assert (got[0] == 0).all() and torch.isfinite(got).all()
        assert (tokens.logprobs_grad(ctx, x, t, r.row_max, r.log_sum, None, g)[4:] == 0).all()
    x = rand(1, 3, v)
    x[0, 0] = NAN
    x[1, 1] = INF
    t = torch.zeros(3, dtype=torch.int64, device="cuda")
    r = tokens.logprobs(ctx, x, t)
    got = tokens.logprobs_grad(ctx, x, t, r.row_max, r.log_sum, r.entropy, g[:3], e[:3])
    assert got[:2].isnan().all() and torch.isfinite(got[2]).all()


def test_logprobs_grad_against_differences(ctx):
    x, t = margins(11, 6, 40, F32)
    t = t.clamp(0, 39)
    g, e, scale = rand(3, 6), rand(4, 6), 0.8
    r = tokens.logprobs(ctx, x, t, scale=scale)
    got = tokens.logprobs_grad(ctx, x, t, r.row_max, r.log_sum, r.entropy, g, e, scale=scale)

    def objective(y):
        _, _, _, logp, ent, _, _, _ = logprob_reference(y, t, scale, 0)
        return g.double() * logp + e.double() * ent
    step = 1e-4
    for j in range(40):
        up, down = x.double().clone(), x.double().clone()
        up[:, j] += step
        down[:, j] -= step
        slope = (objective(up) - objective(down)) / (2 * step)
        # the difference's own error is of the order step^2 and 1e-15 / step
        assert ((slope - got[:, j].double()).abs() < 1e-6).all()


# ---- together ----------------------------------------------------------------------------------


def chain(ctx, table, ids, w, target, weights, seed, dtype):
    """Embedding, dropout, a product, the loss and all their gradients, as a training step
    runs them; returns the outputs and dtable, dw."""
    n, d = ids.numel(), table.shape[1]
    x = tokens.embed(ctx, table, ids, scale=math.sqrt(d), dtype=dtype)
    xd = tokens.dropout(ctx, x, 0.2, seed, 1)
    z = xd @ w
    r = tokens.logprobs(ctx, z, target, top_k=3)
    dz = tokens.logprobs_grad(ctx, z, target, r.row_max, r.log_sum, r.entropy, weights, 0.1 * weights)
    dx = tokens.dropout(ctx, dz @ w.t(), 0.2, seed, 1)
    dtable = tokens.embed_grad(ctx, dx.reshape(n, d), ids, table.shape[0], scale=math.sqrt(d))
    return r, dtable, xd.t() @ dz


def chain_inputs(n=300, vocab=70, d=32, classes=50):
    ids = rand_ids(1, n, vocab)
    table, w = rand(2, vocab, d, std=0.05), rand(3, d, classes, std=0.3)
    target = torch.randint(-1, classes, (n,), device="cuda", generator=torch.Generator("cuda").manual_seed(4))
    weights = -torch.rand(n, device="cuda", generator=torch.Generator("cuda").manual_seed(5))
    return table, ids, w, target, weights


def test_training_step_gradients(ctx):
    """The chain's gradients against 64-bit autograd of the same loss."""
    table, ids, w, target, weights = chain_inputs()
    old = torch.backends.cuda.matmul.allow_tf32
    torch.backends.cuda.matmul.allow_tf32 = False
    try:
        r, dtable, dw = chain(ctx, table, ids, w, target, weights, 9, F32)
    finally:
        torch.backends.cuda.matmul.allow_tf32 = old
    T, W = table.double().requires_grad_(), w.double().requires_grad_()
    seen = (ids >= 0) & (ids < 70)
    x = torch.where(seen[:, None], T[ids.clamp(0, 69)] * math.sqrt(32), 0.0)
    keep = torch.from_numpy(philox_keep(x.numel(), 0.2, 9, 1)).cuda().reshape(x.shape)
    x = torch.where(keep, x * (65536.0 / (65536 - round(0.2 * 65536))), 0.0)
    lp = torch.log_softmax(x @ W, 1)
    logp = torch.where(target >= 0, lp.gather(1, target.clamp(min=0)[:, None])[:, 0], 0.0)
    ent = -(lp.exp() * lp).sum(1)
    (weights.double() * logp + 0.1 * weights.double() * ent).sum().backward()
    # sums of 32 products, then of up to 300 rows, of terms near 1: a few hundred roundings
    assert (r.logp.double() - logp).abs().max() < 200 * U * 10
    assert (dtable.double() - T.grad).abs().max() < 1000 * U * float(T.grad.abs().max() + 1)
    assert (dw.double() - W.grad).abs().max() < 1000 * U * float(W.grad.abs().max() + 1)
    assert (dtable[torch.bincount(ids[seen], minlength=70) == 0] == 0).all()


@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
def test_training_step_in_a_graph(ctx, dtype):
    """Captured and replayed on new inputs, twice, with two graphs alive at once."""
    table, ids, w, target, weights = chain_inputs(n=5000, vocab=900, d=64, classes=1500)
    table, w = table.to(dtype), w.to(dtype)
    graphs = []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        chain(ctx, table, ids, w, target, weights, 9, dtype)
    torch.cuda.current_stream().wait_stream(side)
    for seed in (9, 10):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = chain(ctx, table, ids, w, target, weights, seed, dtype)
        graphs.append((seed, graph, out))
    for change in (1, 2):
        ids.copy_(rand_ids(change, 5000, 900))
        table.copy_(rand(change, 900, 64, std=0.05).to(dtype))
        for _, graph, _ in graphs:
            graph.replay()
        for seed, _, (r, dtable, dw) in graphs:
            q, et, ew = chain(ctx, table, ids, w, target, weights, seed, dtype)
            assert all(torch.equal(a, b) for a, b in zip(r, q))
            assert torch.equal(dtable, et) and torch.equal(dw, ew)


def test_gradient_of_a_column_in_a_graph(ctx):
    """The path without a sort, captured and replayed on new ids."""
    ids, grad = rand_ids(1, 40000, 30), rand(2, 40000, 24)
    out = torch.zeros(30, 24, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        tokens.embed_grad(ctx, grad, ids, 30, out=out)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tokens.embed_grad(ctx, grad, ids, 30, out=out, accumulate=True)
    ids.copy_(rand_ids(3, 40000, 30))
    out.fill_(1.0)
    graph.replay()
    check_grad(out, grad, ids, 30, 1.0, torch.ones_like(out))


def test_two_streams_at_once(ctx):
    """The same calls on two streams, without ordering between them, agree with one."""
    jobs = []
    for i in range(2):
        ids = rand_ids(i, 30000, 500)
        grad = rand(i, 30000, 96)
        x, t = margins(i, 40, 60000, BF16)
        jobs.append((ids, grad, x, t))

    def work(ids, grad, x, t):
        return (tokens.embed_grad(ctx, grad, ids, 500), *tokens.logprobs(ctx, x, t, top_k=8),
                tokens.dropout(ctx, grad, 0.3, 5))
    want = [work(*j) for j in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    got = [None, None]
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = work(*jobs[i])
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_own_stream_of_the_context(ctx):
    """A call on the context's own stream, through the C entry point."""
    x = rand(1, 100, 8)
    y = torch.empty_like(x)
    torch.cuda.synchronize()
    s = N.lib.rw_ctx_stream(ctx.h)
    ctx.check(N.lib.rw_dropout_device(ctx.h, x.data_ptr(), N.RW_F32, 100, 8, 8, 0.5, 1, 2,
                                      y.data_ptr(), 8, s))
    torch.cuda.synchronize()
    assert torch.equal(y, tokens.dropout(ctx, x, 0.5, 1, 2))


def guarded(bytes_needed):
    """A workspace of exactly that many bytes, of all ones, between bytes that must stay."""
    buf = torch.full((bytes_needed + 512,), 255, device="cuda", dtype=torch.uint8)
    return buf, buf[256:256 + bytes_needed], (lambda: bool((buf[:256] == 255).all() and (buf[256 + bytes_needed:] == 255).all()))


@pytest.mark.parametrize("n,d,vocab", [(700, 33, 40), (700, 40, 2000), (30000, 33, 40), (30000, 33, 4000),
                                       (30000, 128, 300), (9, 3, 2)])
def test_embed_grad_workspace_contents_do_not_matter(ctx, n, d, vocab):
    """Through the C entry point: any contents, no byte outside it, no byte between rows."""
    import ctypes as C
    ids, grad = rand_ids(n, n, vocab), rand(n, n, d)
    want = tokens.embed_grad(ctx, grad, ids, vocab)
    need = C.c_uint64()
    ctx.check(N.lib.rw_embed_grad_workspace(ctx.h, n, d, vocab, C.byref(need)))
    buf, ws, fine = guarded(need.value)
    out = torch.full((vocab, d + 5), 3.0, device="cuda")
    ctx.check(N.lib.rw_embed_grad_device(ctx.h, grad.data_ptr(), N.RW_F32, d, ids.data_ptr(), N.RW_I64, n, d,
                                         vocab, 1.0, 0, out.data_ptr(), N.RW_F32, d + 5, ws.data_ptr(),
                                         need.value, torch.cuda.current_stream().cuda_stream))
    assert torch.equal(out[:, :d], want) and (out[:, d:] == 3).all() and fine()


@pytest.mark.parametrize("n,v", [(1, 128000), (8, 50001), (100, 20000), (3, 9000)])
def test_logprobs_workspace_contents_do_not_matter(ctx, n, v):
    import ctypes as C
    x, t = margins(v, n, v, BF16)
    want = tokens.logprobs(ctx, x, t, top_k=32)
    need = C.c_uint64()
    ctx.check(N.lib.rw_logprobs_workspace(ctx.h, n, v, N.RW_BF16, 32, C.byref(need)))
    assert need.value > 0
    buf, ws, fine = guarded(need.value)
    row = torch.full((5, n), 3.0, device="cuda")
    top, index = torch.full((n, 32), 3.0, device="cuda"), torch.full((n, 32), 3, device="cuda")
    ctx.check(N.lib.rw_logprobs_device(ctx.h, x.data_ptr(), N.RW_BF16, n, v, v, 1.0, t.data_ptr(), N.RW_I64, 32,
                                       *(r.data_ptr() for r in row), top.data_ptr(), index.data_ptr(),
                                       ws.data_ptr(), need.value, torch.cuda.current_stream().cuda_stream))
    assert all(torch.equal(a, b) for a, b in zip((*row, top, index), want)) and fine()


@pytest.mark.parametrize("v", [7, 2000])
def test_logprobs_outputs_may_be_left_out(ctx, v):
    x, t = margins(v, 40, v, F32)
    want = tokens.logprobs(ctx, x, t, top_k=3)
    s = torch.cuda.current_stream().cuda_stream
    need = 1 << 20
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    full = [want.row_max, want.log_sum, want.lse, want.logp, want.entropy, want.top_logp, want.top_index]
    for keep in range(7):
        outs = [torch.empty_like(f) if i == keep else None for i, f in enumerate(full)]
        ctx.check(N.lib.rw_logprobs_device(ctx.h, x.data_ptr(), N.RW_F32, 40, v, v, 1.0,
                                           t.data_ptr() if keep == 3 else None, N.RW_I64, 3,
                                           *(None if o is None else o.data_ptr() for o in outs),
                                           ws.data_ptr(), need, s))
        # without the entropy's sum the exponentials are the same; only summation order may not be
        assert torch.allclose(outs[keep].double(), full[keep].double(), rtol=1e-6, atol=1e-6)


def test_strided_outputs_keep_what_lies_between(ctx):
    x = rand(1, 50, 3000)
    t = torch.zeros(50, dtype=torch.int64, device="cuda")
    r = tokens.logprobs(ctx, x, t)
    for call in (lambda o: tokens.dropout(ctx, x, 0.5, 1, out=o),
                 lambda o: tokens.logprobs_grad(ctx, x, t, r.row_max, r.log_sum, None, -r.lse, out=o),
                 lambda o: tokens.dropout(ctx, x, 1.0, 1, out=o)):
        buf = torch.full((50, 3011), 7.0, device="cuda")
        call(buf[:, 5:3005])
        assert (buf[:, :5] == 7).all() and (buf[:, 3005:] == 7).all()


@pytest.mark.parametrize("n,d,vocab", [(30000, 128, 300), (30000, 40, 2000), (9000, 264, 40), (3000, 96, 70)])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_embed_grad_bits_do_not_depend_on_strides(ctx, n, d, vocab, dtype):
    """The sums' order comes from ids, sizes and type where the ids are sorted."""
    ids, grad = rand_ids(n, n, vocab), rand(n, n, d, dtype=dtype)
    want = tokens.embed_grad(ctx, grad, ids, vocab)
    out = strided(torch.zeros(vocab, d, device="cuda"), extra=5)
    for g in (grad, strided(grad, extra=3), strided(grad, extra=1)):
        assert torch.equal(tokens.embed_grad(ctx, g, ids, vocab), want)
        assert torch.equal(tokens.embed_grad(ctx, g, ids, vocab, out=out), want)


def far_rows(v, dtype, scale):
    """Rows whose margins are far from 0 in units of 1 / scale, wholly or in part."""
    at = torch.arange(v, device="cuda")
    x, _ = margins(v, 1, v, dtype)
    x = x.float()[0]
    rows = []
    for mask in (-1e9, -1e10, -1e12, -1e18, -1e20, -1e29, -9e29, -1e31):
        rows.append(torch.full_like(x, mask))
        rows.append(torch.where(at < v * 3 // 4, mask, x))            # the first classes masked
        rows.append(torch.where(at // 8 % 256 < 200, mask, x))        # long runs, whole threads' shares
        rows.append(torch.where(at == v // 2, -mask, x))              # one far above
    level = at.remainder(3).float()
    for top in (1e4, 2.9e6, 3.0e6, 2.3e7, 1.1e9, 1e10, -1e4, -2.9e6, -3.1e6, -1e10):
        near = top / scale
        rows.append(near + level * abs(near) * 2.0 ** -7)             # steps that every type has
        rows.append(near + (at == v - 1).float() * abs(near))         # one class ahead at the end
    rows = torch.stack(rows)
    if dtype == F16:
        rows = rows.clamp(-65504, 65504)
    return rows.to(dtype)


@pytest.mark.parametrize("v", [7, 100, 900, 1500, 30000, 140000])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_logprobs_of_far_finite_margins(ctx, v, dtype):
    """Masks by finite numbers, offsets shared by a row, scales that make margins far."""
    for scale in (1.0, 2.0 ** -10, 1e3, 1e6):
        x = far_rows(v, dtype, scale)
        t = torch.arange(len(x), device="cuda") * 977 % v
        got = tokens.logprobs(ctx, x, t, scale=scale, top_k=2)
        check_logprobs(got, x, t, scale, 2)
        other = tokens.logprobs(ctx, strided(x), t, scale=scale)
        check_logprobs(other, x, t, scale, 0)
        if v in (1500, 30000):  # rows enough that none is split
            many = tokens.logprobs(ctx, x.repeat(12, 1), t.repeat(12), scale=scale, top_k=2)
            check_logprobs(type(many)(*(f[-len(x):] for f in many)), x, t, scale, 2)


def check_scaled_grad(got, *args):
    """check_logprobs_grad for gradients that a 16-bit type may not hold: near its largest number
    and beyond, only the sign and that it is large. Probabilities below 2^-126, f32's smallest
    normal number, may count as 0; there |log p| is near 88 (where it is above 100, what is lost
    is less still), so that loses at most 2^-126 (|g| + |e| (100 + h)) scale."""
    want, tol = grad_of_logprobs(*args)
    h, g, e, scale = args[4:]
    tol = tol + (scale * 2.0 ** -126 * (g.double().abs() + e.double().abs() * (100 + h.double().abs())))[:, None]
    large = want.abs() > torch.finfo(got.dtype).max * 0.98
    tol = tol + half_step(got.dtype) * (want.abs() + tol) + (2.0 ** -25 if got.dtype == F16 else 1e-37)
    off = (got.double() - want).abs()
    assert (large | (off <= tol)).all(), float((off - tol)[~large].max())
    assert ((got.double() * want.sign()) >= torch.finfo(got.dtype).max * 0.95)[large].all()


@pytest.mark.parametrize("v", [7, 100, 900, 1500, 30000, 140000])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_logprobs_grad_of_far_finite_margins(ctx, v, dtype):
    for scale in (1.0, 2.0 ** -10, 1e3):
        x = far_rows(v, dtype, scale)
        t = torch.arange(len(x), device="cuda") * 977 % v
        m, log_sum, _, _, h = (f.float() for f in logprob_reference(x, t, scale, 0)[:5])
        g, e = -torch.ones(len(x), device="cuda"), torch.full((len(x),), 0.5, device="cuda")
        for out in (torch.zeros_like(x), strided(torch.zeros_like(x))):
            tokens.logprobs_grad(ctx, x, t, m, log_sum, h, g, e, scale=scale, out=out)
            check_scaled_grad(out, x, t, m, log_sum, h, g, e, scale)
        got = tokens.logprobs_grad(ctx, x, t, m, log_sum, None, g, scale=scale)
        check_scaled_grad(got, x, t, m, log_sum, h, g, torch.zeros_like(g), scale)


@pytest.mark.parametrize("scale", [1.0, 30.0, 1e3, 1e5, 1e6, 1e12])
@pytest.mark.parametrize("v", [7, 600, 5000, 9001])
def test_entropy_gradient_of_masked_classes_at_large_scales(ctx, v, scale):
    """Few and many classes, by vectors and element by element (a dx that lies differently);
    margins of order 1 / scale, so that many classes count, and of order 1."""
    for dtype in TYPES:
        x, t = margins(v, 6, v, dtype, std=2.0)
        x[:4] = (x[:4].float() / scale).to(dtype)
        t = torch.tensor([v - 1, -1, 2, v - 1, 1, v - 1], device="cuda")
        x[0, : v // 2] = -INF
        x[1, 1:] = -INF
        x[2, 1::2] = -INF
        x[4, 2:] = -INF
        x[5, ::3] = -INF
        m, log_sum, _, _, h = (f.float() for f in logprob_reference(x, t, scale, 0)[:5])
        g = -torch.ones(6, device="cuda")
        gone = x == -INF
        gone[torch.arange(6, device="cuda"), t] = False
        for e in (torch.full((6,), 1e-2, device="cuda"), torch.full((6,), -655.0, device="cuda")):
            for out in (torch.zeros_like(x), strided(torch.zeros_like(x))):
                tokens.logprobs_grad(ctx, x, t, m, log_sum, h, g, e, scale=scale, out=out)
                check_scaled_grad(out, x, t, m, log_sum, h, g, e, scale)
                assert (out[gone] == 0).all()
                tokens.logprobs_grad(ctx, x, None, m, log_sum, h, None, e, scale=scale, out=out)
                check_scaled_grad(out, x, t, m, log_sum, h, torch.zeros_like(g), e, scale)


@pytest.mark.parametrize("v", [7, 900, 30000])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_logprobs_grad_of_far_finite_margins_at_a_large_scale(ctx, v, dtype):
    scale = 1e6
    x = far_rows(v, dtype, scale)
    t = torch.arange(len(x), device="cuda") * 977 % v
    m, log_sum, _, _, h = (f.float() for f in logprob_reference(x, t, scale, 0)[:5])
    g, e = -torch.ones(len(x), device="cuda"), torch.full((len(x),), 0.5, device="cuda")
    for out in (torch.zeros_like(x), strided(torch.zeros_like(x))):
        tokens.logprobs_grad(ctx, x, t, m, log_sum, h, g, e, scale=scale, out=out)
        check_scaled_grad(out, x, t, m, log_sum, h, g, e, scale)


def test_nan_at_the_first_class_ranks_first(ctx):
    """Also where the largest margins are more than are kept as candidates, in few threads."""
    v, k = 140000, 5
    x, _ = margins(1, 1, v, F32)
    at = torch.arange(v, device="cuda")
    x[0] += torch.where(at // 4 % 256 < 4, 30.0, 0.0)
    want = torch.sort(x[0], descending=True, stable=True).indices[:k]
    want = torch.cat([want.new_zeros(1), want[want != 0]])[:k]
    x[0, 0] = NAN
    for n in (1, 600):
        got = tokens.logprobs(ctx, x.expand(n, v).contiguous(), top_k=k)
        assert torch.equal(got.top_index, want.expand(n, k))
        assert got.top_logp.isnan().all()
