"""Sampling from given random numbers (decode.Sampler) against the definition in 64 bits.

The library draws by whole-number weights of 32 bits, from exponentials in fp32 (relative error below 2^-21
for the arguments that keep a weight: a rounded difference and quotient of size up to 23, and the
exponential): a cumulative share can be off by 2^-21 and by 2^-33 a token, less than 2^-12 2^-1 = 1.3e-4 for
2^20 tokens and 1e-6 for the vocabularies drawn here. A token is accepted if its stretch of the cumulative
kept weight, widened by 1e-6, holds the random number; the kept set's edge may move by a token whose
cumulative share is within 1e-6 of top-p. Wherever neither is near, the token is the definition's.
"""
import math

import pytest

pytestmark = pytest.mark.gpu

NEAR = 1e-6


def log(*what):
    print(*what, flush=True)


def ranked(torch, logits, t):
    l = torch.where(logits.isnan(), -math.inf, logits.double())
    order = torch.sort(l, descending=True, stable=True)[1]
    if l[order[0]] == math.inf:
        w = (l == math.inf).double()
    else:
        w = torch.exp((l - l[order[0]]) / t)
    return order, w


def accepted(torch, logits, t, k, p, m, u):
    """{token: its log chances} that the definition and the tolerance allow."""
    l = torch.where(logits.isnan(), -math.inf, logits.double())
    if l.max() == -math.inf:
        return {-1: [-math.inf]}
    order, w = ranked(torch, logits, t if t > 0 else 1.0)
    if not t > 0:
        return {int(order[0]): [0.0]}
    n = len(order) if k <= 0 else min(k, len(order))
    kept_w = w[order[:n]]
    before = (torch.cumsum(kept_w, 0) - kept_w) / kept_w.sum()
    floor = kept_w >= m * (1 - NEAR)
    out = {}
    for slack in ((0.0,) if p >= 1 else (0.0, NEAR, -NEAR)):
        keep = floor & ((before < p + slack) if p < 1 else torch.ones_like(floor))
        keep[0] = True
        ids = order[:n][keep].sort()[0]
        share = torch.cumsum(w[ids], 0) / w[ids].sum()
        low = torch.cat([torch.zeros(1, dtype=torch.float64), share[:-1]])
        for i in ((low - NEAR <= u) & (u < share + NEAR) & (w[ids] > 0)).nonzero()[:, 0].tolist():
            out.setdefault(int(ids[i]), []).append(float(torch.log(w[ids[i]] / w[ids].sum())))
    return out


def run(torch, logits, uniform, t=None, k=None, p=None, m=None):
    from leanstream_amd import decode

    rows = logits.shape[0]
    tokens = torch.full((rows,), -5, dtype=torch.int32, device="cuda")
    logprob = torch.full((rows,), math.nan, device="cuda")

    def f(x, dtype=torch.float32):
        return None if x is None else torch.tensor(x, dtype=dtype, device="cuda")

    call = decode.Sampler(logits, f(uniform), tokens, logprob, f(t), f(k, torch.int32), f(p), f(m))
    call.enqueue()
    torch.cuda.synchronize()
    first, first_log = tokens.clone(), logprob.clone()
    for _ in range(3):      # the same bits again
        tokens.fill_(-5)
        call.enqueue()
        torch.cuda.synchronize()
        assert torch.equal(tokens, first) and torch.equal(logprob, first_log)
    return tokens.tolist(), logprob.tolist()


def check(torch, logits, uniform, t=None, k=None, p=None, m=None):
    rows = logits.shape[0]
    tokens, logs = run(torch, logits, uniform, t, k, p, m)
    f32 = torch.float32
    for r in range(rows):
        args = [1.0 if t is None else t[r], 0 if k is None else k[r], 1.0 if p is None else p[r], 0.0 if m is None else m[r],
                uniform[r]]
        args = [float(torch.tensor(x, dtype=f32)) if i != 1 else x for i, x in enumerate(args)]
        ok = accepted(torch, logits[r].cpu(), *args)
        assert tokens[r] in ok, (r, tokens[r], ok, args)
        wants = ok[tokens[r]]
        assert any(logs[r] == x or abs(logs[r] - x) <= 1e-5 + 1e-6 * abs(x) for x in wants), (r, logs[r], wants)


def random_rows(torch, rows, vocab, dtype, seed, peaks=12, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    l = torch.randn(rows, vocab, generator=g) * spread
    at = torch.randint(0, vocab, (rows, min(peaks, vocab)), generator=g)
    l.scatter_add_(1, at, 4 + 6 * torch.rand(at.shape, generator=g))
    u = torch.rand(rows, generator=g).tolist()
    return l.to(getattr(torch, dtype)).cuda(), u, g


@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("vocab", [1, 2, 5, 63, 1000, 4096, 8191, 32768, 50257, 131072])
def test_settings_row_by_row(torch_gpu, vocab, dtype):
    torch = torch_gpu
    rows = 24
    log("case:", vocab, dtype)
    logits, u, g = random_rows(torch, rows, vocab, dtype, vocab)
    r = list(range(rows))
    t = [[0.7, 1.0, 1.3, 0.0][i % 4] for i in r]
    k = [[0, 1, 2, 50, 40, vocab, vocab + 9, -3][i % 8] for i in r]
    p = [[1.0, 0.9, 0.5, 0.1, 0.99][i % 5] for i in r]
    m = [[0.0, 0.05, 0.3][i % 3] for i in r]
    check(torch, logits, u, t, k, p, m)
    check(torch, logits, u, t)
    check(torch, logits, u, None, k)
    check(torch, logits, u, None, None, p)
    check(torch, logits, u, None, None, None, m)


@pytest.mark.parametrize("rows,vocab", [(1, 200000), (1, 1 << 20), (3, 1 << 20), (300, 777)])
def test_large_and_many(torch_gpu, rows, vocab):
    torch = torch_gpu
    logits, u, g = random_rows(torch, rows, vocab, "bfloat16", rows + vocab)
    check(torch, logits, u, [0.8] * rows, None, [0.95] * rows)
    check(torch, logits, u, [0.8] * rows, [100] * rows)
    check(torch, logits, u, [1.5] * rows)


def test_flat_rows_keep_the_lowest_ids(torch_gpu):
    """Equal logits are ranked by id: k of them are the first k, and top-p takes the first ones too."""
    torch = torch_gpu
    vocab = 5000
    logits = torch.zeros(6, vocab, device="cuda")
    logits[:, ::2] = 1.0        # 2500 tokens with the same best logit
    u = [0.0, 0.5, 0.999999, 0.25, 0.75, 0.9]
    tokens, _ = run(torch, logits, u, None, [10, 10, 10, 2500, 2499, 2600])
    assert tokens[:3] == [0, 10, 18]
    check(torch, logits, u, None, [10, 10, 10, 2500, 2499, 2600])
    check(torch, logits, u, None, [100] * 6, [0.5, 0.333, 0.1, 0.999, 0.01, 0.0])
    check(torch, logits, u, None, None, [0.5, 0.333, 0.1, 0.999, 0.01, 0.73])
    flat = torch.full((4, 131072), -3.25, dtype=torch.float16, device="cuda")
    check(torch, flat, [0.0, 0.3, 0.7, 0.99], None, [1000, 5, 0, 70000], [1.0, 0.5, 0.5, 0.1])


def test_ties_at_the_cut_among_others(torch_gpu):
    """Few distinct logits, many tokens of each: the cut falls into a run of equal ones."""
    torch = torch_gpu
    g = torch.Generator().manual_seed(5)
    logits = torch.randint(0, 8, (16, 30000), generator=g).half().cuda()
    u = torch.rand(16, generator=g).tolist()
    check(torch, logits, u, None, [1 + 977 * i for i in range(16)])
    check(torch, logits, u, [2.0] * 16, [20000] * 16, [0.05 + 0.06 * i for i in range(16)])


def test_infinities_nan_and_empty_rows(torch_gpu):
    torch = torch_gpu
    inf, nan = math.inf, math.nan
    logits = torch.randn(8, 300, device="cuda")
    logits[0] = -inf
    logits[1] = nan
    logits[2, :299] = -inf
    logits[3, 100:] = nan
    logits[4, [7, 90, 200]] = inf
    logits[5] = torch.finfo(torch.float32).min
    logits[5, 17] = 0.0
    logits[6] = torch.finfo(torch.float32).min
    logits[7, 5] = torch.finfo(torch.float32).max
    u = [0.5, 0.5, 0.9, 0.7, 0.5, 0.99, 0.5, 0.3]
    for t in (None, [0.7] * 8, [0.0] * 8):
        for k, p in ((None, None), ([5] * 8, [0.9] * 8)):
            check(torch, logits, u, t, k, p)
    tokens, logs = run(torch, logits, u)
    assert tokens[:3] == [-1, -1, 299] and logs[0] == -inf and logs[2] == 0.0
    assert tokens[4] == 90 and tokens[5] == 17 and tokens[7] == 5


def test_extreme_settings(torch_gpu):
    """Numbers at and beyond the ends of their ranges."""
    torch = torch_gpu
    logits, _, _ = random_rows(torch, 8, 1000, "float32", 3)
    best = logits.argmax(1).tolist()
    u = [0.0, 1.0 - 2.0 ** -24, 0.0, 0.5, 0.5, 0.5, 0.5, 0.5]
    check(torch, logits, u)
    for p in (0.0, -1.0, 1e-30):
        assert run(torch, logits, u, None, None, [p] * 8)[0] == best
    for m in (1.0, 2.0):
        assert run(torch, logits, u, None, None, None, [m] * 8)[0] == best
    assert run(torch, logits, u, [1e-30] * 8)[0] == best
    assert run(torch, logits, u, [-1.0] * 8)[0] == best
    assert run(torch, logits, u, [math.nan] * 8)[0] == best
    check(torch, logits, u, None, None, [2.0] * 8)
    tokens, _ = run(torch, logits, [math.nan, -1.0, 1.0, 2.0, math.inf, -math.inf, 0.5, 0.5])
    assert all(0 <= x < 1000 for x in tokens)
    # every logit counts alike at an infinite temperature
    check(torch, logits, u, [math.inf] * 8)


@pytest.mark.parametrize("dtype", ["float16", "float32"])
def test_many_infinite_logits(torch_gpu, dtype):
    """More infinite logits than a chunk has room for, at any temperature: they share the row."""
    torch = torch_gpu
    logits, u, g = random_rows(torch, 4, 20000, dtype, 8)
    for r, n in enumerate((300, 6000, 20000, 1)):
        logits[r, torch.randperm(20000, generator=g)[:n]] = math.inf
    for t in (None, [math.inf] * 4, [1e-6] * 4):
        for k, p, m in (([10] * 4, None, None), (None, [0.5] * 4, None), ([400] * 4, [0.9] * 4, None), (None, None, [0.5] * 4)):
            check(torch, logits, u, t, k, p, m)


def test_neighbouring_logits_at_tiny_temperatures(torch_gpu):
    """Logits a unit in the last place apart, of weights that still compare, many of each."""
    torch = torch_gpu
    near = 10.0 - 2.0 ** -20
    g = torch.Generator().manual_seed(12)
    logits = torch.randn(4, 20000, generator=g)
    for r, (few, many) in enumerate(((10, 6000), (1, 8000), (100, 250), (3, 15000))):
        at = torch.randperm(20000, generator=g)
        logits[r, at[:few]] = 10.0
        logits[r, at[few:few + many]] = near
    u = torch.rand(4, generator=g).tolist()
    for k, p, m in (([20] * 4, None, None), (None, [0.5] * 4, None), ([400] * 4, [0.9] * 4, None), (None, None, [0.3] * 4)):
        check(torch, logits.cuda(), u, [1e-6] * 4, k, p, m)


def test_rows_of_any_stride_and_alignment(torch_gpu):
    torch = torch_gpu
    for dtype in (torch.float16, torch.float32):
        wide = torch.randn(5, 40007, device="cuda").mul(3).to(dtype)
        for begin, vocab in ((0, 40007), (1, 40000), (3, 33333), (8, 1024)):
            logits = wide[:, begin:begin + vocab]
            check(torch, logits, [0.1, 0.3, 0.5, 0.7, 0.9], None, [64] * 5, [0.9] * 5)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("vocab", [3000, 20000, 60001, 131072])
def test_wide_nuclei(torch_gpu, vocab, dtype):
    """Rows without outstanding tokens: top-p keeps thousands (in bf16 many of them equal), with and without a
    min-p that keeps fewer; top-k beyond what a chunk remembers."""
    torch = torch_gpu
    rows = 12
    logits, u, g = random_rows(torch, rows, vocab, dtype, vocab + 1, peaks=1, spread=1.0)
    p = [0.2, 0.5, 0.8, 0.9, 0.95, 0.99, 0.999, 0.3, 0.6, 0.7, 0.97, 0.9]
    check(torch, logits, u, None, None, p)
    check(torch, logits, u, [3.0] * rows, None, p)
    check(torch, logits, u, [0.2, 0.5, 1.7, 30.0] * 3, None, p)
    check(torch, logits, u, [2.0] * rows, None, p, [0.001, 0.05, 0.3] * 4)
    check(torch, logits, u, [2.0] * rows, [2999, 1500, 700] * 4, p)
    check(torch, logits, u, [2.0] * rows, [2999, 1500, 700] * 4)
    check(torch, logits, u, [2.0] * rows, None, None, [0.001, 0.05, 0.3] * 4)
