"""The operators around the MLP of a decode step, as their speed is measured.

A case is one call that a serving loop makes once a layer or once a step: the attention of new
tokens over a paged cache (`attention`), the rotation of q and k and the write of k and v into
the cache's pages (`append`), the norms and the residual between two blocks (`norm`), and the
pick of the next tokens (`sample`).
"""
import math
import random

import torch

own = False

DEV = "cuda"
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
MAX_FLOPS = 2.2e12      # of a drawn attention case: the largest listed one
MAX_BYTES = 1.1e9       # of any drawn case


def _attention(name, dtype, heads, kv_heads, dim, page, seqs, context, new=1, chunks=0, window=0, sinks=0, mix=1):
    """`seqs` sequences of up to `context` keys; the first `chunks` of them bring up to `new` tokens,
    the others one each. `mix` seeds the lengths."""
    c = dict(kind="attention", dtype=dtype, heads=heads, kv_heads=kv_heads, dim=dim, page=page, seqs=seqs,
             context=context, new=new, chunks=chunks, window=window, sinks=sinks, mix=mix)
    return dict(c, name=name) if name else c


def _append(name, dtype, heads, kv_heads, dim, rot, page, seqs, context, new=1, chunks=0, interleaved=False, mix=1):
    c = dict(kind="append", dtype=dtype, heads=heads, kv_heads=kv_heads, dim=dim, rot=rot, page=page, seqs=seqs,
             context=context, new=new, chunks=chunks, interleaved=interleaved, mix=mix)
    return dict(c, name=name) if name else c


def _norm(name, dtype, rows, width, post=True, gate="none", offset=0.0, scale=1.0):
    c = dict(kind="norm", dtype=dtype, rows=rows, width=width, post=post, gate=gate, offset=offset, scale=scale)
    return dict(c, name=name) if name else c


def _sample(name, dtype, rows, vocab, style):
    c = dict(kind="sample", dtype=dtype, rows=rows, vocab=vocab, style=style)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one sequence's next token over a short cache: the smallest call, where latency counts (8B-model heads)
        _attention("attn_one", "fp16", 32, 8, 128, 16, 1, 777),
        # batched decode, ragged contexts, 70B-model heads
        _attention("attn_b32", "bf16", 64, 8, 128, 16, 32, 8192, mix=2),
        # decode of two long documents
        _attention("attn_long", "fp16", 32, 8, 128, 64, 2, 131072, mix=3),
        # a prompt's last chunk over everything before it: the largest call
        _attention("attn_chunk", "fp16", 32, 8, 128, 64, 1, 32768, new=4096, chunks=1),
        # a serving step that mixes prompt chunks with decodes, window and sink tokens, a head each
        _attention("attn_mixed", "bf16", 16, 16, 64, 32, 24, 16384, new=512, chunks=3, window=4096, sinks=4, mix=4),
        # the new tokens of 32 sequences go into the cache
        _append("append_b32", "fp16", 32, 8, 128, 128, 16, 32, 1024, mix=5),
        # a prompt's chunk goes into the cache, adjacent pairs, half of the dimensions rotated
        _append("append_chunk", "bf16", 64, 8, 128, 64, 64, 1, 12288, new=8192, chunks=1, interleaved=True),
        # between two blocks of a decode step, one sequence
        _norm("norm_one", "fp16", 1, 4096),
        # between two blocks of a prompt's chunk, a gate for every element, weights stored around zero
        _norm("norm_chunk", "bf16", 8192, 8192, gate="full", offset=1.0, scale=0.5),
        # one sequence's next token: temperature and top-p
        _sample("sample_one", "fp16", 1, 32768, "top_p"),
        # a batch whose requests each bring their own settings, some of them greedy
        _sample("sample_b64", "bf16", 64, 131072, "mixed"),
        # many requests, full-precision logits, an odd vocabulary
        _sample("sample_b256", "fp32", 256, 50257, "top_k"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attention"] * 4 + ["append", "norm", "sample", "sample"])
    dtype = rng.choice(["fp16", "bf16"])
    mix = rng.randint(1, 1 << 30)
    if kind in ("attention", "append"):
        kv = rng.choice([1, 2, 4, 8, 16])
        heads = kv * rng.choice([1, 2, 4, 7, 8] if kv <= 8 else [1, 2])
        dim = rng.choice([64, 128, 128, 256])
        page = rng.choice([1, 16, 16, 32, 64, 128])
        seqs = _log(rng, 1, 64)
        while True:
            context = _log(rng, 1, 131072 if kind == "attention" else 8192)
            new = min(context, _log(rng, 1, 4096))
            chunks = rng.choice([0, 0, 1, rng.randint(1, seqs)])
            if kind == "attention":
                window = rng.choice([0, 0, _log(rng, 16, 8192)])
                c = _attention(None, dtype, heads, kv, dim, page, seqs, context, new if chunks else 1, chunks, window,
                               rng.choice([0, 4, 7]) if window else 0, mix)
            else:
                c = _append(None, dtype, heads, kv, dim, rng.choice([dim, dim, dim // 2]), page, seqs, context,
                            new if chunks else 1, chunks, rng.choice([False, False, True]), mix)
            w = work(c)
            if w["flops"] <= MAX_FLOPS and w["bytes"] <= MAX_BYTES and \
                    2 * seqs * _pages_each(c) * page * kv * dim * 2 <= 2 * MAX_BYTES:
                return c
            seqs = max(1, seqs // 2)
    if kind == "norm":
        width = rng.choice([1024, 4096, 8192, _log(rng, 33, 16384)])
        return _norm(None, rng.choice([dtype, dtype, "fp32"]), _log(rng, 1, min(8192, 60000000 // width)), width,
                     rng.choice([True, True, False]), rng.choice(["none", "shared", "full"]), rng.choice([0.0, 1.0]),
                     rng.choice([1.0, 0.25]))
    vocab = rng.choice([32768, 131072, _log(rng, 300, 200000)])
    return _sample(None, rng.choice([dtype, "fp32"]), _log(rng, 1, min(256, 16000000 // vocab)), vocab,
                   rng.choice(["top_p", "top_k", "min_p", "mixed"]))


# ---------------------------------------------------------------------------- lengths
def _lengths(case):
    """(new tokens, keys with them) of every sequence. Of many sequences the last is an idle slot."""
    rng = random.Random(case["mix"])
    out = []
    for s in range(case["seqs"]):
        if s < case["chunks"]:
            new = case["new"] if s == 0 else rng.randint(1, case["new"])
        else:
            new = 1
        keys = case["context"] if s == 0 else rng.randint(max(1, case["context"] // 4), case["context"])
        out.append((min(new, keys), keys))
    if case["seqs"] > 8:
        out[-1] = (0, 0)
    return out


def _pages_each(case):
    return -(-case["context"] // case["page"])


def _pairs(new, keys, window, sinks):
    """Visible (token, key) pairs of a sequence, and the keys that any of its tokens sees."""
    first = keys - new
    if not window:
        return new * (2 * first + new + 1) // 2, keys if new else 0
    pairs = 0
    for p in range(first, keys):
        low = max(0, p + 1 - window)
        pairs += p + 1 - low + min(sinks, low)
    low = max(0, first + 1 - window)
    return pairs, (keys - low + min(sinks, low)) if new else 0


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    kind = case["kind"]
    if kind in ("attention", "append"):
        lengths = _lengths(case)
        tokens = sum(n for n, _ in lengths)
        row = case["dim"] * size
        if kind == "append":
            wide = 2 * (case["heads"] + 2 * case["kv_heads"]) * row
            return {"bytes": tokens * (wide + case["rot"] * 4), "flops": tokens * 3 * (case["heads"] + case["kv_heads"]) *
                    case["rot"]}
        pairs = keys = 0
        for n, k in lengths:
            p, u = _pairs(n, k, case["window"], case["sinks"])
            pairs, keys = pairs + p, keys + u
        return {"bytes": 2 * tokens * case["heads"] * row + 2 * keys * case["kv_heads"] * row,
                "flops": 4 * case["dim"] * case["heads"] * pairs}
    if kind == "norm":
        n = case["rows"] * case["width"]
        wide = 4 + (case["gate"] == "full")
        return {"bytes": n * wide * size + 3 * case["width"] * size, "flops": n * 10}
    n = case["rows"] * case["vocab"]
    return {"bytes": n * size + 28 * case["rows"], "flops": n * 4}


# ---------------------------------------------------------------------------- inputs
def _gen(seed, what, device=DEV):
    return torch.Generator(device=device).manual_seed(1000003 * int(seed) + what)


def _randn(shape, seed, what, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, device=DEV, generator=_gen(seed, what)) * scale).to(dtype)


def _sequences(case, seed):
    """Lengths, start of every sequence's tokens and a table of pages in random order, -1 where a
    sequence holds no page (past its end, or behind its window)."""
    lengths = _lengths(case)
    starts = [0]
    for n, _ in lengths:
        starts.append(starts[-1] + n)
    each, page = _pages_each(case), case["page"]
    pages = case["seqs"] * each
    table = torch.randperm(pages, generator=_gen(seed, 1, "cpu")).to(torch.int32).view(case["seqs"], each)
    window, sinks = case.get("window", 0), case.get("sinks", 0)
    for s, (n, k) in enumerate(lengths):
        table[s, -(-k // page):] = -1
        if window:
            gone = max(0, k - n + 1 - window) // page          # pages wholly behind every token's window
            table[s, -(-sinks // page):max(gone, -(-sinks // page))] = -1
    return dict(lengths=lengths, starts=starts, pages=pages, table=table.to(DEV),
                q_start=torch.tensor(starts, dtype=torch.int32, device=DEV),
                context=torch.tensor([k for _, k in lengths], dtype=torch.int32, device=DEV))


def _inputs(case, seed):
    dtype = TYPES[case["dtype"]]
    kind = case["kind"]
    if kind in ("attention", "append"):
        st = _sequences(case, seed)
        H, K, D, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
        tokens = st["starts"][-1]
        shape = (st["pages"], K, page, D)
        # keys with a common direction and queries that favour it: some keys weigh more, as in a trained model
        st["k_pages"] = _randn(shape, seed, 2, dtype, 1.25)
        st["v_pages"] = _randn(shape, seed, 3, dtype)
        if kind == "attention":
            st["q"] = _randn((tokens, H, D), seed, 4, dtype, 1.5)
            st["out"] = torch.empty_like(st["q"])
            st["scale"] = D ** -0.5
        else:
            # one projection gives q, k and v of a token side by side
            qkv = _randn((tokens, (H + 2 * K) * D), seed, 4, dtype).view(tokens, H + 2 * K, D)
            st["q"], st["k"], st["v"] = qkv[:, :H], qkv[:, H:H + K], qkv[:, H + K:]
            st["q_out"] = torch.empty(tokens, H, D, dtype=dtype, device=DEV)
            half = case["rot"] // 2
            inv = 1e6 ** (-torch.arange(half, dtype=torch.float64) / half)
            angle = torch.arange(case["context"], dtype=torch.float64)[:, None] * inv
            st["cos"], st["sin"] = torch.cos(angle).float().to(DEV), torch.sin(angle).float().to(DEV)
        return st
    if kind == "norm":
        R, d = case["rows"], case["width"]
        st = dict(block=_randn((R, d), seed, 1, dtype, 0.7), residual=_randn((R, d), seed, 2, dtype, 2.0))
        mean = 1.0 - case["offset"]
        st["pre"] = (mean + 0.1 * torch.randn(d, device=DEV, generator=_gen(seed, 3))).to(dtype)
        st["post"] = (mean + 0.1 * torch.randn(d, device=DEV, generator=_gen(seed, 4))).to(dtype) if case["post"] else None
        st["gate"] = None
        if case["gate"] != "none":
            st["gate"] = _randn((R, d) if case["gate"] == "full" else (d,), seed, 5, dtype, 0.5)
        st["hidden"], st["normed"] = torch.empty_like(st["block"]), torch.empty_like(st["block"])
        st["eps"] = 1e-5
        return st
    R, V = case["rows"], case["vocab"]
    logits = torch.randn(R, V, device=DEV, generator=_gen(seed, 1)) * 2.0
    # a few tokens of every row stand out, as a trained model's do
    top = torch.randint(0, V, (R, 24), device=DEV, generator=_gen(seed, 2))
    logits.scatter_add_(1, top, 5.0 + 6.0 * torch.rand(R, 24, device=DEV, generator=_gen(seed, 3)))
    g = _gen(seed, 4, "cpu")
    temperature = 0.6 + 0.6 * torch.rand(R, generator=g)
    top_k = torch.randint(20, 201, (R,), generator=g, dtype=torch.int32)
    top_p = 0.8 + 0.15 * torch.rand(R, generator=g)
    min_p = 0.02 + 0.08 * torch.rand(R, generator=g)
    which = torch.arange(R) % 5 if case["style"] == "mixed" else torch.full((R,), ["top_p", "top_k", "min_p"].index(
        case["style"]))
    # of "mixed": top-p, top-k, min-p, all three, greedy
    top_p = torch.where((which == 0) | (which == 3), top_p, 1.0)
    top_k = torch.where((which == 1) | (which == 3), top_k, 0).to(torch.int32)
    min_p = torch.where((which == 2) | (which == 3), min_p, 0.0)
    temperature = torch.where(which == 4, 0.0, temperature)
    return dict(logits=logits.to(dtype), temperature=temperature.to(DEV), top_k=top_k.to(DEV), top_p=top_p.to(DEV),
                min_p=min_p.to(DEV), uniform=torch.rand(R, device=DEV, generator=_gen(seed, 5)),
                tokens=torch.empty(R, dtype=torch.int32, device=DEV), logprob=torch.empty(R, device=DEV))


def prepare(case, seed):
    st = _inputs(case, seed)
    st["case"] = case
    if not own:
        return st
    from leanstream_amd import decode

    kind = case["kind"]
    if kind in ("attention", "append"):
        cache = decode.PagedCache(st["k_pages"], st["v_pages"])
        max_new = max(n for n, _ in st["lengths"])
    if kind == "attention":
        st["call"] = decode.PagedAttention(st["q"], cache, st["table"], st["q_start"], st["context"], st["out"],
                                           max_new=max_new, max_context=case["context"], scale=st["scale"],
                                           window=case["window"], sinks=case["sinks"])
    elif kind == "append":
        st["call"] = decode.AppendKV(st["q"], st["k"], st["v"], st["cos"], st["sin"], cache, st["table"], st["q_start"],
                                     st["context"], st["q_out"], interleaved=case["interleaved"])
    elif kind == "norm":
        st["call"] = decode.BlockNorm(st["block"], st["residual"], st["hidden"], st["normed"], pre_weight=st["pre"],
                                      post_weight=st["post"], gate=st["gate"], residual_scale=case["scale"],
                                      weight_offset=case["offset"], eps=st["eps"])
    else:
        st["call"] = decode.Sampler(st["logits"], st["uniform"], st["tokens"], st["logprob"],
                                    temperature=st["temperature"], top_k=st["top_k"], top_p=st["top_p"],
                                    min_p=st["min_p"])
    return st


def run(st):
    case = st["case"]
    kind = case["kind"]
    if own:
        st["call"].enqueue()
        return {"attention": lambda: st["out"], "append": lambda: [st["q_out"], st["k_pages"], st["v_pages"]],
                "norm": lambda: [st["hidden"], st["normed"]],
                "sample": lambda: [st["tokens"], st["logprob"]]}[kind]()
    return {"attention": _plain_attention, "append": _plain_append, "norm": _plain_norm,
            "sample": _plain_sample}[kind](case, st)


# ---------------------------------------------------------------------------- plain forms (32 bits)
def _visible(pos, keys, window, sinks):
    """[tokens, keys] truth values: key positions that a token at pos sees."""
    j = torch.arange(keys, device=DEV)
    see = j[None, :] <= pos[:, None]
    if window:
        see &= (j[None, :] > pos[:, None] - window) | (j[None, :] < sinks)
    return see


def _plain_attention(case, st):
    H, K, page = case["heads"], case["kv_heads"], case["page"]
    G = H // K
    out = torch.zeros_like(st["q"])
    for s, (n, keys) in enumerate(st["lengths"]):
        if not n:
            continue
        t0 = st["starts"][s]
        ids = st["table"][s, :-(-keys // page)].clamp(min=0).long()
        # [K, keys, D]
        k = st["k_pages"][ids].transpose(0, 1).flatten(1, 2)[:, :keys]
        v = st["v_pages"][ids].transpose(0, 1).flatten(1, 2)[:, :keys]
        step = max(1, (1 << 28) // (G * keys))
        for a in range(0, n, step):
            b = min(n, a + step)
            pos = torch.arange(keys - n + a, keys - n + b, device=DEV)
            see = _visible(pos, keys, case["window"], case["sinks"]).repeat_interleave(G, 0)
            for h in range(K):
                q = st["q"][t0 + a:t0 + b, h * G:(h + 1) * G].reshape((b - a) * G, -1).float()
                score = (q @ k[h].float().t()) * st["scale"]
                score.masked_fill_(~see, -math.inf)
                top = score.amax(1, keepdim=True)
                p = torch.exp(score - top.clamp(min=-1e30))
                o = (p @ v[h].float()) / p.sum(1, keepdim=True).clamp(min=1e-30)
                out[t0 + a:t0 + b, h * G:(h + 1) * G] = o.view(b - a, G, -1).to(out.dtype)
    return out


def _positions(st):
    seq, pos = [], []
    for s, (n, keys) in enumerate(st["lengths"]):
        seq.append(torch.full((n,), s, device=DEV))
        pos.append(torch.arange(keys - n, keys, device=DEV))
    return torch.cat(seq), torch.cat(pos)


def _rotate(x, cos, sin, rot, interleaved):
    """x [tokens, heads, D]; cos, sin [tokens, rot / 2]."""
    c, s = cos[:, None], sin[:, None]
    y = x.clone()
    if interleaved:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y[..., 0:rot:2], y[..., 1:rot:2] = a * c - b * s, b * c + a * s
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y[..., :rot // 2], y[..., rot // 2:rot] = a * c - b * s, b * c + a * s
    return y


def _plain_append(case, st):
    seq, pos = _positions(st)
    page = case["page"]
    ids, slot = st["table"][seq, pos // page].long(), pos % page
    cos, sin = st["cos"][pos], st["sin"][pos]
    dtype = st["q"].dtype
    st["q_out"].copy_(_rotate(st["q"].float(), cos, sin, case["rot"], case["interleaved"]).to(dtype))
    k = _rotate(st["k"].float(), cos, sin, case["rot"], case["interleaved"]).to(dtype)
    st["k_pages"][ids, :, slot] = k
    st["v_pages"][ids, :, slot] = st["v"]
    return [st["q_out"], st["k_pages"], st["v_pages"]]


def _plain_norm(case, st):
    y = st["block"].float()
    if st["post"] is not None:
        y = y / torch.sqrt((y * y).mean(1, keepdim=True) + st["eps"]) * (case["offset"] + st["post"].float())
    if st["gate"] is not None:
        y = y * st["gate"].float()
    h = case["scale"] * st["residual"].float() + y
    n = h / torch.sqrt((h * h).mean(1, keepdim=True) + st["eps"]) * (case["offset"] + st["pre"].float())
    return [h.to(st["block"].dtype), n.to(st["block"].dtype)]


def _share(total, fraction, up):
    """total * fraction rounded down (or up) in whole numbers; the fraction in steps of 2^-24."""
    m = (fraction.double() * 16777216.0).long()
    high, low = total >> 24, total & 16777215
    return m * high + ((m * low + (16777215 if up else 0)) >> 24)


def _plain_sample(case, st):
    l = st["logits"].float()
    R, V = l.shape
    t = st["temperature"][:, None]
    greedy = t <= 0
    x = (l - l.amax(1, keepdim=True)) / torch.where(greedy, 1.0, t)
    e = torch.exp(x)
    order = torch.sort(l, dim=1, descending=True, stable=True)[1]
    e_rank = e.gather(1, order)
    w_rank = torch.round(e_rank * 4294967296.0).long()
    rank = torch.arange(V, device=DEV)[None, :]
    top_k = st["top_k"][:, None]
    keep = (top_k <= 0) | (rank < top_k)
    w_k = torch.where(keep, w_rank, 0)
    limit = _share(w_k.sum(1, keepdim=True), st["top_p"][:, None], True).clamp(min=1)
    keep &= (w_k.cumsum(1) - w_k < limit) & (e_rank >= st["min_p"][:, None])
    keep = torch.where(greedy, rank < 1, keep)
    w = torch.zeros(R, V, dtype=torch.int64, device=DEV).scatter_(1, order, torch.where(keep, w_rank, 0))
    total = w.sum(1, keepdim=True)
    token = (w.cumsum(1) <= _share(total, st["uniform"][:, None], False)).sum(1, keepdim=True)
    logprob = torch.log(w.gather(1, token).float() / total.float())
    return [token[:, 0].to(torch.int32), logprob[:, 0]]


# ---------------------------------------------------------------------------- definition in 64 bits
def exact(case, seed):
    st = _inputs(case, seed)
    return {"attention": _exact_attention, "append": _exact_append, "norm": _exact_norm,
            "sample": _exact_sample}[case["kind"]](case, st)


def _exact_attention(case, st):
    G, page = case["heads"] // case["kv_heads"], case["page"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=DEV)
    token = 0
    for s, (n, keys) in enumerate(st["lengths"]):
        for a in range(0, n, 512):
            count = min(512, n - a)
            where = torch.arange(keys - n + a, keys - n + a + count, device=DEV)
            # the keys that this block of tokens can see at all
            j = torch.arange(int(where[-1]) + 1, device=DEV)
            if case["window"]:
                j = j[(j > int(where[0]) - case["window"]) | (j < case["sinks"])]
            hidden = j[None] > where[:, None]
            if case["window"]:
                hidden |= (where[:, None] - j[None] >= case["window"]) & (j[None] >= case["sinks"])
            at = st["table"][s, j // page].long()
            for h in range(case["heads"]):
                key = st["k_pages"][at, h // G, j % page].double()
                value = st["v_pages"][at, h // G, j % page].double()
                z = st["q"][token + a:token + a + count, h].double().mm(key.t()).mul_(st["scale"])
                z[hidden] = -math.inf
                out[token + a:token + a + count, h] = torch.softmax(z, 1).mm(value)
        token += n
    return out


def _exact_append(case, st):
    k_pages, v_pages = st["k_pages"].double(), st["v_pages"].double()
    q_out = st["q"].double()
    half, page = case["rot"] // 2, case["page"]
    i = torch.arange(half, device=DEV)
    first, second = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + half)
    token = 0
    for s, (n, keys) in enumerate(st["lengths"]):
        if not n:
            continue
        rows = slice(token, token + n)
        p = torch.arange(keys - n, keys, device=DEV)
        turn = torch.complex(st["cos"][p].double(), st["sin"][p].double())[:, None]
        at, slot = st["table"][s, p // page].long(), p % page
        for name in ("q", "k"):
            x = st[name][rows].double()
            z = torch.complex(x[..., first], x[..., second]) * turn
            x[..., first], x[..., second] = z.real, z.imag
            if name == "q":
                q_out[rows] = x
            else:
                k_pages[at, :, slot] = x
        v_pages[at, :, slot] = st["v"][rows].double()
        token += n
    return [q_out, k_pages, v_pages]


def _exact_norm(case, st):
    def unit(x, weight):
        return x * torch.rsqrt(x.pow(2).sum(1, keepdim=True) / case["width"] + st["eps"]) * (weight.double() +
                                                                                             case["offset"])

    z = st["block"].double()
    z = unit(z, st["post"]) if case["post"] else z
    z = z * st["gate"].double() if case["gate"] != "none" else z
    h = st["residual"].double() * case["scale"] + z
    return [h, unit(h, st["pre"])]


def _exact_sample(case, st):
    tokens, logs = [], []
    for r in range(case["rows"]):
        l = st["logits"][r].double()
        t, k, p, m, u = (float(st[name][r]) for name in ("temperature", "top_k", "top_p", "min_p", "uniform"))
        if t <= 0:
            tokens.append(int((l == l.max()).nonzero()[0]))
            logs.append(0.0)
            continue
        chance = torch.softmax(l / t, 0)
        ranked, ids = torch.sort(chance, dim=0, descending=True, stable=True)
        if k > 0:
            ranked, ids = ranked[:int(k)], ids[:int(k)]
        ranked = ranked / ranked.sum()
        nucleus = torch.cumsum(ranked, 0) - ranked < p
        nucleus &= ranked >= m * ranked[0]
        kept = ids[nucleus].sort()[0]
        share = torch.cumsum(chance[kept] / chance[kept].sum(), 0)
        i = min(int((share <= u).sum()), kept.numel() - 1)
        tokens.append(int(kept[i]))
        logs.append(float(torch.log(chance[kept[i]] / chance[kept].sum())))
    return [torch.tensor(tokens, dtype=torch.int32, device=DEV), torch.tensor(logs, dtype=torch.float64, device=DEV)]
