"""The norms between two blocks (decode.BlockNorm) and the cache's new slots (decode.AppendKV) against
their formulas in 64 bits.

Tolerances, per element, with u the unit roundoff of the type: u |x| for the output's rounding and, for the
arithmetic in fp32, 2^-18 of the sum of the terms' sizes (a sum of up to 16384 squares in one accumulator of
64 and a tree, a square root, a division and a few products). A rotation: u |x| + 2^-21 (|a| + |b|).
"""
import math

import pytest

pytestmark = pytest.mark.gpu

U = {"float16": 2.0 ** -11, "bfloat16": 2.0 ** -8, "float32": 2.0 ** -24}


def log(*what):
    print(*what, flush=True)


def rms(x, eps):
    return (x.pow(2).mean(1, keepdim=True) + eps).sqrt()


def norm_expected(block, residual, pre, post, gate, scale, offset, eps):
    """(hidden, normed, sizes of hidden's terms) in float64."""
    z = block.double()
    if post is not None:
        z = z / rms(z, eps) * (offset + post.double())
    if gate is not None:
        z = z * gate.double()
    r = scale * residual.double()
    h = r + z
    return h, h / rms(h, eps) * (offset + pre.double()), r.abs() + z.abs()


SHAPES = [(1, 4096), (3, 8192), (1, 16384), (5, 1), (2, 7), (130, 64), (9, 1000), (4, 4095), (2, 5003), (33, 2048), (1, 10240)]


@pytest.mark.parametrize("dtype", list(U))
@pytest.mark.parametrize("rows,width", SHAPES)
def test_norm_formula(torch_gpu, rows, width, dtype):
    torch = torch_gpu
    from leanstream_amd import decode

    log("case:", rows, width, dtype)
    t, u = getattr(torch, dtype), U[dtype]
    g = torch.Generator().manual_seed(rows * 100003 + width)

    def rand(*shape, mean=0.0, scale=1.0):
        return (mean + scale * torch.randn(*shape, generator=g)).to(t)

    for with_post, gate_kind, scale, offset, eps in [(True, "full", 0.5, 1.0, 1e-5), (False, None, 1.0, 0.0, 1e-6),
                                                     (True, "row", -1.25, 0.0, 1e-5), (False, "full", 1.0, 0.0, 0.5)]:
        block, residual = rand(rows, width, scale=0.7), rand(rows, width, scale=2.0)
        pre, post = rand(width, mean=1.0 - offset, scale=0.1), rand(width, mean=1.0 - offset, scale=0.1) if with_post else None
        gate = None if gate_kind is None else rand(rows, width) if gate_kind == "full" else rand(width)
        h, n, size = norm_expected(block, residual, pre, post, gate, scale, offset, eps)
        hidden, normed = torch.empty(rows, width, dtype=t, device="cuda"), torch.empty(rows, width, dtype=t, device="cuda")
        dev = [x.cuda() if x is not None else None for x in (pre, post, gate)]
        decode.BlockNorm(block.cuda(), residual.cuda(), hidden, normed, dev[0], dev[1], dev[2], scale, offset, eps).enqueue()
        torch.cuda.synchronize()
        factor = (offset + pre.double()).abs() / rms(h, eps)
        assert ((hidden.cpu().double() - h).abs() <= u * h.abs() + 2.0 ** -18 * size).all()
        assert ((normed.cpu().double() - n).abs() <= u * n.abs() + 2.0 ** -18 * size * factor + 1e-45).all()
        # one output alone gives the same bits
        for keep in (True, False):
            alone = torch.empty_like(hidden)
            decode.BlockNorm(block.cuda(), residual.cuda(), alone if keep else None, None if keep else alone, dev[0], dev[1],
                             dev[2], scale, offset, eps).enqueue()
            torch.cuda.synchronize()
            assert torch.equal(alone, hidden if keep else normed)


@pytest.mark.parametrize("dtype", ["float16", "float32"])
@pytest.mark.parametrize("width,offset", [(512, 0), (512, 1), (515, 3), (4096, 8)])
def test_norm_strides_offsets_and_in_place(torch_gpu, width, offset, dtype):
    """Rows in wider tensors, any alignment of an element; hidden over residual, normed over block."""
    torch = torch_gpu
    from leanstream_amd import decode

    t, u, rows = getattr(torch, dtype), U[dtype], 6
    g = torch.Generator().manual_seed(width + offset)
    wide = torch.randn(rows, 3 * width + 2 * offset + 5, generator=g).to(t).cuda()
    block, residual = wide[:, offset:offset + width], wide[:, width + offset + 3:2 * width + offset + 3]
    rest = wide[:, 2 * width + offset + 3:].clone()
    pre = (1 + 0.1 * torch.randn(width + offset, generator=g)).to(t).cuda()[offset:]
    h, n, size = norm_expected(block.cpu(), residual.cpu(), pre.cpu(), pre.cpu(), None, 1.0, 0.0, 1e-5)
    decode.BlockNorm(block, residual, residual, block, pre, pre).enqueue()
    torch.cuda.synchronize()
    factor = pre.cpu().double().abs() / rms(h, 1e-5)
    assert ((residual.cpu().double() - h).abs() <= u * h.abs() + 2.0 ** -18 * size).all()
    assert ((block.cpu().double() - n).abs() <= u * n.abs() + 2.0 ** -18 * size * factor).all()
    assert torch.equal(wide[:, 2 * width + offset + 3:], rest)


def test_norm_rows_are_independent_and_zeros_stay(torch_gpu):
    torch = torch_gpu
    from leanstream_amd import decode

    x = torch.randn(9, 768, device="cuda").half()
    x[3] = math.nan
    x[5] = 0
    w = torch.ones(768, device="cuda").half()
    hidden, normed = torch.empty_like(x), torch.empty_like(x)
    decode.BlockNorm(x, torch.zeros_like(x), hidden, normed, w, w).enqueue()
    torch.cuda.synchronize()
    assert hidden[3].isnan().all() and normed[3].isnan().all()
    assert (normed[5] == 0).all()
    rest = [0, 1, 2, 4, 6, 7, 8]
    assert normed[rest].isfinite().all()


def append_problem(torch, dtype, dim, q_heads, kv_heads, page, lengths, rot, interleaved, order, seed=1):
    g = torch.Generator().manual_seed(seed)
    t = getattr(torch, dtype)
    width = max(1, max(-(-k // page) for _, k in lengths))
    pages = len(lengths) * width + 2
    table = torch.randperm(pages, generator=g)[: len(lengths) * width].to(torch.int32).view(-1, width)
    tokens = sum(n for n, _ in lengths)
    qkv = torch.randn(tokens, q_heads + 2 * kv_heads, dim, generator=g).to(t)
    angle = torch.rand(max(1, max(k for _, k in lengths)), rot // 2, generator=g, dtype=torch.float64) * 6.283
    starts = [0]
    for n, _ in lengths:
        starts.append(starts[-1] + n)
    k = torch.randn(pages, kv_heads, page, dim, generator=g).to(t)
    v = torch.randn(pages, kv_heads, page, dim, generator=g).to(t)
    return dict(table=table, qkv=qkv, cos=angle.cos().float(), sin=angle.sin().float(), starts=starts, k=k, v=v)


def turned(x, cos, sin, rot, interleaved):
    y = x.double().clone()
    tol = y.abs()
    half = rot // 2
    i = list(range(0, rot, 2)) if interleaved else list(range(half))
    j = list(range(1, rot, 2)) if interleaved else list(range(half, rot))
    if rot:
        a, b = y[:, i].clone(), y[:, j].clone()
        y[:, i], y[:, j] = a * cos.double() - b * sin.double(), b * cos.double() + a * sin.double()
        tol[:, i] = tol[:, j] = a.abs() + b.abs()
    return y, tol


APPENDS = [
    dict(dim=128, q_heads=32, kv_heads=8, page=16, lengths=[(1, 1), (1, 17), (0, 5), (1, 500)], rot=128),
    dict(dim=64, q_heads=6, kv_heads=3, page=1, lengths=[(9, 9), (0, 0), (4, 60)], rot=32),
    dict(dim=256, q_heads=4, kv_heads=1, page=64, lengths=[(100, 130), (1, 65)], rot=256),
    dict(dim=96, q_heads=5, kv_heads=5, page=4, lengths=[(33, 40)], rot=96),
    dict(dim=80, q_heads=0, kv_heads=2, page=8, lengths=[(20, 20), (3, 9)], rot=20),
    dict(dim=10, q_heads=3, kv_heads=1, page=32, lengths=[(7, 33)], rot=6),
    dict(dim=128, q_heads=8, kv_heads=2, page=16, lengths=[(21, 50)], rot=0),
]


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("case", range(len(APPENDS)))
def test_append_formula(torch_gpu, case, interleaved, dtype):
    torch = torch_gpu
    from leanstream_amd import decode

    c = APPENDS[case]
    log("case:", case, interleaved, dtype)
    dim, H, K, page, rot, lengths = (c[n] for n in ("dim", "q_heads", "kv_heads", "page", "rot", "lengths"))
    p = append_problem(torch, dtype, **c, interleaved=interleaved, order="head")
    for order in ("head", "slot", "one"):
        k, v = p["k"].cuda(), p["v"].cuda()
        if order == "slot":
            k, v = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (k, v))
        qkv = p["qkv"].cuda()
        if order == "one":    # an odd row length: rows start at any element
            flat = torch.zeros(qkv.shape[0], (H + 2 * K) * dim + 1, dtype=qkv.dtype, device="cuda")
            flat[:, 1:] = qkv.flatten(1)
            qkv = flat[:, 1:].unflatten(1, (H + 2 * K, dim))
        q, kn, vn = qkv[:, :H], qkv[:, H:H + K], qkv[:, H + K:]
        q_out = torch.empty(q.shape, dtype=q.dtype, device="cuda") if order != "one" else q    # in place
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        decode.AppendKV(q if H else None, kn, vn, p["cos"].cuda() if rot else None, p["sin"].cuda() if rot else None,
                        decode.PagedCache(k, v), p["table"].cuda(),
                        torch.tensor(p["starts"], dtype=torch.int32, device="cuda"),
                        torch.tensor([m for _, m in lengths], dtype=torch.int32, device="cuda"), q_out if H else None,
                        interleaved=interleaved, status=status).enqueue()
        torch.cuda.synchronize()
        assert int(status) == 0
        want_k, want_v = p["k"].double(), p["v"].clone()
        tol_k = torch.zeros_like(want_k)
        u = U[dtype]
        for s, (n, keys) in enumerate(lengths):
            for i in range(n):
                pos, t = keys - n + i, p["starts"][s] + i
                at, slot = int(p["table"][s, pos // page]), pos % page
                cos, sin = (p["cos"][pos], p["sin"][pos])
                x, size = turned(p["qkv"][t], cos, sin, rot, interleaved)
                if H:
                    off = (q_out[t].cpu().double() - x[:H]).abs()
                    assert (off <= u * x[:H].abs() + 2.0 ** -21 * size[:H]).all()
                want_k[at, :, slot] = x[H:H + K]
                tol_k[at, :, slot] = u * x[H:H + K].abs() + 2.0 ** -21 * size[H:H + K]
                want_v[at, :, slot] = p["qkv"][t, H + K:]
        assert ((k.cpu().double() - want_k).abs() <= tol_k).all()
        assert torch.equal(v.cpu(), want_v)


def test_append_leaves_out_what_has_no_place(torch_gpu):
    """A negative position, a position beyond the tables, no page: nothing is written but the status."""
    torch = torch_gpu
    from leanstream_amd import decode

    K, dim, page = 2, 64, 16
    for lengths, spoil, want in ([(4, 2)], None, 8), ([(2, 40)], "positions", 8), ([(2, 40)], "page", 4), ([(2, 40)], "width", 8):
        p = append_problem(torch, "float16", dim, 0, K, page, lengths, 64, False, "head")
        k, v = p["k"].cuda(), p["v"].cuda()
        table, cos, sin = p["table"], p["cos"], p["sin"]
        context = [m for _, m in lengths]
        if spoil == "positions":
            cos, sin = cos[:39].contiguous(), sin[:39].contiguous()
        if spoil == "page":
            table = table.clone()
            table[0, 2] = -1
        if spoil == "width":
            context = [10 ** 9]
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        decode.AppendKV(None, p["qkv"][:, :K].cuda(), p["qkv"][:, K:].cuda(), cos.cuda(), sin.cuda(),
                        decode.PagedCache(k, v), table.cuda(), torch.tensor(p["starts"], dtype=torch.int32, device="cuda"),
                        torch.tensor(context, dtype=torch.int32, device="cuda"), None, status=status).enqueue()
        torch.cuda.synchronize()
        assert int(status) == want
        changed = (k.cpu() != p["k"]).flatten(0, 0).any(3).any(1).sum() if spoil != "x" else 0
        assert int(changed) == {None: 2, "positions": 1, "page": 0, "width": 0}[spoil]
