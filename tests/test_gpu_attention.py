"""Attention over a paged cache (leanstream_amd.decode.PagedAttention) against the formula in 64 bits.

Tolerance, per element, with u the unit roundoff of the type (2^-11 for fp16, 2^-8 for bf16) and p the exact
softmax: u |o| for the output's rounding, u sum p |v| for the rounding of p before the second product, 2^-12
sum p |v| for the scores (a sum of up to 256 products in fp32, |q||k| scale of order 10: 256 x 10 x 2^-24) and
the exponentials, and in fp16 half a subnormal step, 2^-25 of the largest p, for every key. The logarithm of
the sum: 2^-12, and 2^-20 of its size.
"""
import math

import pytest

pytestmark = pytest.mark.gpu

U = {"float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


def log(*what):
    print(*what, flush=True)


class Problem:
    """Random inputs on the CPU; `lengths` is [(new tokens, keys)] of every sequence."""

    def __init__(self, torch, dtype, dim, heads, kv_heads, page, lengths, window=0, sinks=0, seed=1, order="head",
                 fill=0.0, spread=1.0):
        self.torch, self.dtype, self.lengths, self.window, self.sinks = torch, getattr(torch, dtype), lengths, window, sinks
        self.u, self.page, self.heads, self.kv_heads, self.dim = U[dtype], page, heads, kv_heads, dim
        g = torch.Generator().manual_seed(seed)
        width = max(1, max(-(-k // page) for _, k in lengths))
        self.pages = len(lengths) * width + 3
        self.table = torch.randperm(self.pages, generator=g)[: len(lengths) * width].to(torch.int32).view(-1, width)
        tokens = sum(n for n, _ in lengths)
        self.q = (torch.randn(tokens, heads, dim, generator=g) * spread).to(self.dtype)
        shape = (self.pages, kv_heads, page, dim)
        self.k = torch.full(shape, fill, dtype=self.dtype)
        self.v = torch.full(shape, fill, dtype=self.dtype)
        for s, (n, keys) in enumerate(lengths):     # what is never written keeps `fill`
            for j in range(0, keys, page):
                m = min(page, keys - j)
                at = int(self.table[s, j // page])
                self.k[at, :, :m] = torch.randn(kv_heads, m, dim, generator=g).to(self.dtype)
                self.v[at, :, :m] = torch.randn(kv_heads, m, dim, generator=g).to(self.dtype)
        self.order = order
        starts = [0]
        for n, _ in lengths:
            starts.append(starts[-1] + n)
        self.starts = starts
        self.scale = dim ** -0.5

    def on_gpu(self, **kw):
        torch = self.torch
        from leanstream_amd import decode

        k, v = self.k.cuda(), self.v.cuda()
        if self.order == "slot":       # memory order [page, slot, head, dim]
            k, v = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (k, v))
        cache = decode.PagedCache(k, v)
        self.q_gpu = self.q.cuda()
        if self.order == "slot":       # q as a part of a wider projection, out head-major
            wide = torch.full((self.q.shape[0], self.heads + 3, self.dim), math.nan, dtype=self.dtype, device="cuda")
            wide[:, 2:2 + self.heads] = self.q_gpu
            self.q_gpu = wide[:, 2:2 + self.heads]
            self.out = torch.full((self.heads, self.q.shape[0], self.dim), math.nan, dtype=self.dtype,
                                  device="cuda").transpose(0, 1)
        else:
            self.out = torch.full(self.q.shape, math.nan, dtype=self.dtype, device="cuda")
        self.lse = torch.full(self.q.shape[:2], math.nan, device="cuda")
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.q_start = torch.tensor(self.starts, dtype=torch.int32, device="cuda")
        self.context = torch.tensor([k for _, k in self.lengths], dtype=torch.int32, device="cuda")
        args = dict(max_new=max(n for n, _ in self.lengths), max_context=max(1, max(k for _, k in self.lengths)),
                    window=self.window, sinks=self.sinks, lse=self.lse, status=self.status, scale=self.scale)
        args.update(kw)
        return decode.PagedAttention(self.q_gpu, cache, self.table.cuda(), self.q_start, self.context, self.out, **args)

    def expected(self):
        """(out, lse, tolerance of out) in float64."""
        torch = self.torch
        out = torch.zeros(self.q.shape, dtype=torch.float64)
        tol = torch.zeros_like(out)
        lse = torch.full(self.q.shape[:2], -math.inf, dtype=torch.float64)
        group = self.heads // self.kv_heads
        for s, (n, keys) in enumerate(self.lengths):
            j = torch.arange(keys)
            at = self.table[s].long()
            k = self.k[at[j // self.page], :, j % self.page].double()
            v = self.v[at[j // self.page], :, j % self.page].double()
            for i in range(n):
                p = keys - n + i
                see = j <= p
                if self.window:
                    see &= (j > p - self.window) | (j < self.sinks)
                if not see.any():
                    continue
                t = self.starts[s] + i
                kk = k[see].repeat_interleave(group, 1)
                vv = v[see].repeat_interleave(group, 1)
                z = (kk * self.q[t].double()).sum(2) * self.scale          # [keys, heads]
                lse[t] = torch.logsumexp(z, 0)
                w = torch.exp(z - lse[t])
                out[t] = (w[..., None] * vv).sum(0)
                weight = (w[..., None] * vv.abs()).sum(0)
                tol[t] = self.u * out[t].abs() + (self.u + 2.0 ** -12) * weight
                if self.dtype == torch.float16:
                    tol[t] += 2.0 ** -25 * int(see.sum()) * w.max(0)[0][:, None] * vv.abs().amax(0)
        return out, lse, tol

    def check(self, status=0):
        self.torch.cuda.synchronize()
        out, lse, tol = self.expected()
        got, got_lse = self.out.cpu().double(), self.lse.cpu().double()
        off = (got - out).abs() - tol
        assert self.torch.isfinite(got).all()
        assert off.max() <= 0, f"out off by {off.max():.3e} more than its tolerance"
        none = lse == -math.inf
        assert bool((got_lse[none] == -math.inf).all()) and bool((got[none] == 0).all())
        assert ((got_lse - lse)[~none].abs() <= 2.0 ** -12 + 2.0 ** -20 * lse[~none].abs()).all()
        assert int(self.status) == status


RAGGED = [(1, 1), (1, 17), (3, 3), (0, 40), (0, 0), (1, 64), (5, 200), (1, 333), (70, 70), (33, 129), (1, 1030)]

CASES = {
    # one token each, from one key on
    "decode": dict(dim=128, heads=32, kv_heads=8, page=16, lengths=[(1, k) for k in (1, 2, 15, 16, 17, 63, 64, 65, 500, 1500)]),
    "decode_mqa": dict(dim=128, heads=16, kv_heads=1, page=32, lengths=[(1, 700), (1, 31), (1, 2049)]),
    "decode_mqa_wide": dict(dim=64, heads=40, kv_heads=1, page=16, lengths=[(1, 900), (1, 5)]),
    "decode_mha": dict(dim=64, heads=6, kv_heads=6, page=16, lengths=[(1, 77), (1, 1300)]),
    "few_tokens": dict(dim=128, heads=8, kv_heads=2, page=64, lengths=[(4, 400), (2, 2), (3, 1025), (1, 64)]),
    "ragged": dict(dim=128, heads=8, kv_heads=2, page=16, lengths=RAGGED),
    "ragged_64": dict(dim=64, heads=6, kv_heads=3, page=8, lengths=RAGGED),
    "ragged_256": dict(dim=256, heads=4, kv_heads=2, page=32, lengths=RAGGED),
    "group_of_7": dict(dim=128, heads=14, kv_heads=2, page=16, lengths=RAGGED),
    "page_1": dict(dim=128, heads=4, kv_heads=1, page=1, lengths=[(1, 77), (20, 130), (1, 3)]),
    "page_2": dict(dim=64, heads=4, kv_heads=2, page=2, lengths=[(1, 77), (20, 130), (1, 300)]),
    "page_4_256": dict(dim=256, heads=4, kv_heads=2, page=4, lengths=[(1, 77), (9, 130), (1, 300)]),
    "page_512": dict(dim=128, heads=8, kv_heads=2, page=512, lengths=[(1, 1100), (40, 600)]),
    "chunk": dict(dim=128, heads=8, kv_heads=2, page=64, lengths=[(300, 900)]),
    "chunk_more_tokens_than_keys": dict(dim=128, heads=4, kv_heads=2, page=16, lengths=[(50, 20), (3, 1), (2, 0)]),
    "window": dict(dim=128, heads=8, kv_heads=2, page=16, lengths=RAGGED, window=50),
    "window_1": dict(dim=64, heads=8, kv_heads=2, page=16, lengths=RAGGED, window=1),
    "window_sinks": dict(dim=128, heads=8, kv_heads=2, page=16, lengths=RAGGED + [(200, 900), (1, 2500)], window=100, sinks=4),
    "window_sinks_wide": dict(dim=64, heads=4, kv_heads=4, page=32, lengths=RAGGED + [(90, 700)], window=33, sinks=150),
    "window_longer_than_all": dict(dim=128, heads=8, kv_heads=2, page=16, lengths=RAGGED, window=5000, sinks=7),
}


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("name", CASES)
def test_formula(torch_gpu, name, dtype):
    log("case:", name, dtype)
    p = Problem(torch_gpu, dtype, **CASES[name])
    p.on_gpu().enqueue()
    p.check()


@pytest.mark.parametrize("name", ["ragged", "window_sinks", "ragged_256", "few_tokens"])
def test_other_orders_and_strides(torch_gpu, name):
    log("case:", name)
    p = Problem(torch_gpu, "bfloat16", **CASES[name], order="slot")
    p.on_gpu().enqueue()
    p.check()


def test_large_scores(torch_gpu):
    """Scores of +-100 and more: all weight on few keys, most others far below the smallest fp16."""
    for dtype in ("float16", "bfloat16"):
        p = Problem(torch_gpu, dtype, 128, 8, 2, 16, [(1, 700), (40, 300)], spread=40.0)
        p.on_gpu().enqueue()
        torch_gpu.cuda.synchronize()
        out, _, tol = p.expected()
        # the scores' fp32 sums are 40 times larger here, and so is their share of the tolerance
        off = (p.out.cpu().double() - out).abs() - 41 * tol
        assert off.max() <= 0


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf, 65504.0])
@pytest.mark.parametrize("name", ["decode", "ragged", "ragged_64", "ragged_256", "window_sinks", "page_1"])
def test_what_slots_hold_that_no_token_sees(torch_gpu, name, bad):
    """Slots past every sequence's end, and whole unwritten pages."""
    log("case:", name, bad)
    p = Problem(torch_gpu, "float16", **CASES[name], fill=bad)
    p.on_gpu().enqueue()
    p.check()


@pytest.mark.parametrize("dim,heads,kv_heads,n", [(128, 8, 2, 40), (64, 4, 4, 150), (256, 4, 2, 20), (128, 8, 2, 4), (64, 8, 1, 2)])
@pytest.mark.parametrize("dtype,bad", [("float16", math.inf), ("float16", math.nan), ("bfloat16", math.nan)])
def test_later_tokens_do_not_reach_earlier_ones(torch_gpu, dim, heads, kv_heads, n, dtype, bad):
    """The last key and value of a chunk are not finite: only the tokens that see them are."""
    p = Problem(torch_gpu, dtype, dim, heads, kv_heads, 16, [(n, 300)])
    at, slot = int(p.table[0, 299 // 16]), 299 % 16
    p.k[at, :, slot] = bad
    p.v[at, :, slot, ::3] = bad
    p.on_gpu().enqueue()
    torch_gpu.cuda.synchronize()
    got = p.out.cpu().double()
    p.k[at, :, slot] = 0
    p.v[at, :, slot] = 0
    out, _, tol = p.expected()
    assert ((got - out).abs() <= tol)[:-1].all()
    assert got[-1].isnan().any()


def test_behind_the_window_is_not_read(torch_gpu):
    """Pages that every token's window has left are gone: their entries are no pages, and what is still in
    partly visible ones is not finite."""
    torch = torch_gpu
    for dim, n in ((128, 1), (128, 60), (64, 3), (256, 1)):
        p = Problem(torch, "float16", dim, 4, 2, 16, [(n, 1000), (n, 150)], window=40, sinks=5)
        want = p.expected()
        for s, (n_, keys) in enumerate(p.lengths):
            low = keys - n_ + 1 - 40
            for j in range(5, max(5, low)):
                at = int(p.table[s, j // 16])
                p.k[at, :, j % 16], p.v[at, :, j % 16] = math.nan, math.inf
        table = p.table.clone()
        for s, (n_, keys) in enumerate(p.lengths):
            gone = max(0, keys - n_ + 1 - 40) // 16
            table[s, 1:gone] = torch.tensor([-1, 1 << 30, p.pages])[torch.arange(1, max(1, gone)) % 3].to(torch.int32)
            table[s, -(-keys // 16):] = -7
        p.table, keep = table, p.table
        p.on_gpu().enqueue()
        p.table = keep
        p.expected = lambda: want
        p.check()


def test_bad_lengths_and_pages_raise_the_status(torch_gpu):
    torch = torch_gpu
    for name in ("decode", "few_tokens", "chunk"):
        # a visible page that does not exist
        p = Problem(torch, "float16", **CASES[name])
        p.table[0, 0] = p.pages
        p.on_gpu().enqueue()
        torch.cuda.synchronize()
        assert int(p.status) == 4
        # a context beyond its bound: that sequence has no keys, the others are as ever
        p = Problem(torch, "float16", **CASES[name])
        call = p.on_gpu()
        p.context[0] += 100000
        call.enqueue()
        p.lengths = [(p.lengths[0][0], 0)] + p.lengths[1:]
        p.check(status=8)
        # tokens out of range: nothing is written for them
        p = Problem(torch, "float16", **CASES[name])
        call = p.on_gpu()
        p.q_start[-1] += 1000
        call.enqueue()
        torch.cuda.synchronize()
        assert int(p.status) == 8
        assert p.out[p.starts[-2]:].isnan().all()


def test_long_cache_past_32_bits(torch_gpu):
    """Pages beyond 2^32 elements (keys and values share the tensor), decode and chunk."""
    torch = torch_gpu
    from leanstream_amd import decode

    page, kv, dim, heads, keys = 64, 8, 128, 16, 300
    each = page * kv * dim
    pages = (1 << 32) // each + 64
    store = torch.empty(pages, kv, page, dim, dtype=torch.float16, device="cuda")
    width = -(-keys // page)
    g = torch.Generator().manual_seed(3)
    data = torch.randn(width, kv, page, dim, generator=g).half()
    ids = torch.arange(pages - width, pages)
    store[ids.cuda()] = data.cuda()
    for n in (1, 30):
        p = Problem(torch, "float16", dim, heads, kv, page, [(n, keys)])
        p.k = p.v = data
        p.table = torch.arange(width, dtype=torch.int32)[None]
        out = torch.empty(p.q.shape, dtype=torch.float16, device="cuda")
        call = decode.PagedAttention(p.q.cuda(), decode.PagedCache(store, store), ids.to(torch.int32)[None].cuda(),
                                     torch.tensor([0, n], dtype=torch.int32, device="cuda"),
                                     torch.tensor([keys], dtype=torch.int32, device="cuda"), out, max_new=n,
                                     max_context=keys)
        call.enqueue()
        torch.cuda.synchronize()
        want, _, tol = p.expected()
        assert ((out.cpu().double() - want).abs() <= tol).all()


@pytest.mark.parametrize("name", ["decode", "few_tokens", "ragged", "window_sinks"])
def test_repeats_give_the_same_bits(torch_gpu, name):
    torch = torch_gpu
    p = Problem(torch, "bfloat16", **CASES[name])
    call = p.on_gpu()
    call.enqueue()
    torch.cuda.synchronize()
    first, first_lse = p.out.clone(), p.lse.clone()
    for _ in range(4):
        p.out.fill_(math.nan)
        call.enqueue()
        torch.cuda.synchronize()
        assert torch.equal(p.out, first) and torch.equal(p.lse, first_lse)


def test_wrong_tensors_are_refused(torch_gpu):
    torch = torch_gpu
    p = Problem(torch, "float16", **CASES["few_tokens"])
    with pytest.raises(RuntimeError, match="Native attention failed: 22"):
        p.on_gpu(max_context=100000).enqueue()
    long = Problem(torch, "float16", **CASES["decode"])
    call = long.on_gpu(workspace=torch.zeros(16, dtype=torch.uint8, device="cuda"))
    with pytest.raises(RuntimeError, match="Native attention failed: 28"):
        call.enqueue()
    with pytest.raises(ValueError, match="float16"):
        p.q = p.q.float()
        p.on_gpu()


def test_workspaces_and_bounds_that_do_not_fit_are_refused(torch_gpu):
    """Decided when the call is bound: a workspace off the GPU or of other elements, numbers beyond 32 bits."""
    torch = torch_gpu
    p = Problem(torch, "float16", **CASES["few_tokens"])
    with pytest.raises(ValueError, match="off the GPU"):
        p.on_gpu(workspace=torch.zeros(1 << 20, dtype=torch.uint8))
    with pytest.raises(ValueError, match="bytes"):
        p.on_gpu(workspace=torch.zeros(1 << 20, device="cuda"))
    for name in ("window", "sinks", "max_new", "max_context"):
        for value in (-1, 1 << 30, (1 << 32) + 8):
            with pytest.raises(ValueError, match="lie in"):
                p.on_gpu(**{name: value})


def test_one_workspace_for_calls_of_every_shape(torch_gpu):
    """Calls that follow one another on a stream share a workspace, whatever each leaves in it."""
    torch = torch_gpu
    names = ["decode", "ragged", "few_tokens", "chunk", "decode_mqa", "window_sinks", "decode"]
    problems = [Problem(torch, "float16", **CASES[n]) for n in names]
    need = max(p.on_gpu().workspace.numel() if p.on_gpu().workspace is not None else 0 for p in problems)
    shared = torch.zeros(need, dtype=torch.uint8, device="cuda")
    calls = [p.on_gpu(workspace=shared) for p in problems]
    for _ in range(2):
        for c in calls:
            c.enqueue()
    for p in problems:
        p.check()


def test_a_workspace_after_calls_without_row_splits(torch_gpu):
    """A call that only splits tiles leaves the counters of later calls' splits alone."""
    torch = torch_gpu
    chunk = Problem(torch, "bfloat16", 64, 40, 1, 16, [(30, 2000), (17, 900)])    # no sequence of few rows
    one = Problem(torch, "bfloat16", 128, 8, 2, 16, [(1, 6000)])
    need = max(p.on_gpu().workspace.numel() for p in (chunk, one))
    shared = torch.zeros(need, dtype=torch.uint8, device="cuda")
    calls = [p.on_gpu(workspace=shared) for p in (chunk, one)]
    for _ in range(2):
        for c in calls:
            c.enqueue()
    for p in (chunk, one):
        p.check()


def test_long_split_sequences(torch_gpu):
    """Many splits of few rows and of tiles: one long sequence alone, and long ones among short ones."""
    torch = torch_gpu
    for dim, heads, kv, lengths in ((128, 4, 1, [(1, 20000)]), (64, 2, 2, [(3, 9000), (1, 40)]), (128, 8, 2, [(40, 7000)]),
                                    (64, 4, 4, [(150, 3000), (1, 5000), (20, 6000)]), (256, 4, 1, [(1, 6000), (30, 5000)])):
        for window, sinks in ((0, 0), (2500, 9)):
            log("case:", dim, heads, lengths, window)
            p = Problem(torch, "float16", dim, heads, kv, 32, lengths, window=window, sinks=sinks)
            p.on_gpu().enqueue()
            p.check()


def test_values_that_are_not_finite_in_split_tiles(torch_gpu):
    """As above, where the last tile's keys are a split of their own."""
    torch = torch_gpu
    p = Problem(torch, "float16", 128, 8, 2, 16, [(40, 3000)])
    at, slot = int(p.table[0, 2990 // 16]), 2990 % 16
    p.v[at, 1, slot, 5] = math.inf       # seen by the last 10 tokens, by heads 4 .. 7
    p.on_gpu().enqueue()
    torch.cuda.synchronize()
    got = p.out.cpu().double()
    assert (got[30:, 4:, 5] == math.inf).all()
    got[30:, 4:, 5] = 0
    p.v[at, 1, slot, 5] = 0
    out, _, tol = p.expected()
    out[30:, 4:, 5] = 0
    # that value's weight (below 1 / 100 of a row here) is not missed elsewhere
    assert ((got - out).abs() <= tol).all()
