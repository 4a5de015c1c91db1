"""A small decoder around the streamed MLP: prompts in one chunk, then a token of every sequence a step.

    python -m leanstream_amd.decode_step

Every layer is norm -> q, k, v projection -> rotary positions and cache append -> paged attention -> output
projection -> norm -> sparse INT4 MLP (the resident layer of ls_hip_core_layer_noalloc) -> norm, and the last
hidden states go through a vocabulary projection and the sampler. The projections are plain matrix products;
everything else is this library's. Weights are random: the example shows how the calls fit together, and which
buffers a program keeps.
"""
import numpy as np
import torch

from . import _native, decode, synth

DEV = "cuda"


class Decoder:
    """Weights and caches of `layers` layers. `bind(tokens, max_new)` gives the step for that many tokens a call."""

    def __init__(self, layers=2, width=1024, q_heads=16, kv_heads=4, head_dim=64, groups=64, active=16, vocab=2048,
                 sequences=4, max_context=256, page_size=16, window=0, sinks=0, seed=1):
        g = torch.Generator(device=DEV).manual_seed(seed)

        def rand(*shape, scale=1.0, mean=0.0):
            return (mean + scale * torch.randn(shape, device=DEV, generator=g)).half()

        self.width, self.q_heads, self.kv_heads, self.head_dim, self.vocab = width, q_heads, kv_heads, head_dim, vocab
        self.sequences, self.max_context, self.window, self.sinks = sequences, max_context, window, sinks
        self.embedding = rand(vocab, width)
        self.head = rand(width, vocab, scale=width ** -0.5)
        self.last_norm = rand(width, scale=0.1, mean=1.0)
        each = -(-max_context // page_size)
        self.page_table = torch.randperm(sequences * each, device=DEV, generator=g).to(torch.int32).view(sequences, each)
        angle = torch.arange(max_context, dtype=torch.float64)[:, None] * 1e4 ** (
            -torch.arange(head_dim // 2, dtype=torch.float64) / (head_dim // 2))
        self.cos, self.sin = angle.cos().float().to(DEV), angle.sin().float().to(DEV)
        self.groups, group_bytes = groups, 64 * 3 * width // 2
        cfg = synth.LayerConfig("decode_step", width, groups * 64, active / groups)
        core = synth.descriptors(cfg, np.arange(active) * groups // active)
        self.core, self.core_count = torch.from_numpy(core.astype(np.int32)).to(DEV), active
        self.layers = [dict(
            attention_norm=rand(width, scale=0.1, mean=1.0), mlp_norm=rand(width, scale=0.1, mean=1.0),
            after_mlp=rand(width, scale=0.1, mean=1.0), gate=rand(width, scale=0.1, mean=0.5),
            qkv=rand(width, (q_heads + 2 * kv_heads) * head_dim, scale=width ** -0.5),
            out=rand(q_heads * head_dim, width, scale=(q_heads * head_dim) ** -0.5),
            mlp=torch.randint(0, 256, (groups * group_bytes,), dtype=torch.uint8, device=DEV, generator=g),
            mlp_scales=(0.001 + 0.002 * torch.rand(groups * 64 * 3 * (width // 128), device=DEV, generator=g)).half(),
            cache=decode.PagedCache.empty(sequences * each, kv_heads, page_size, head_dim, torch.float16),
        ) for _ in range(layers)]

    def bind(self, tokens, max_new):
        return Step(self, tokens, max_new)


class Step:
    """The calls of one step over `tokens` tokens, bound once; `run` fills their inputs and enqueues them."""

    def __init__(self, decoder, tokens, max_new):
        d = self.decoder = decoder
        self.tokens, self.max_new = tokens, max_new

        def buffer(*shape, dtype=torch.float16):
            return torch.empty(shape, dtype=dtype, device=DEV)

        self.q_start = buffer(d.sequences + 1, dtype=torch.int32)
        self.context = buffer(d.sequences, dtype=torch.int32)
        self.status = torch.zeros(1, dtype=torch.int32, device=DEV)
        self.hidden, self.normed = buffer(tokens, d.width), buffer(tokens, d.width)
        self.qkv = buffer(tokens, d.q_heads + 2 * d.kv_heads, d.head_dim)
        self.rotated, self.attended = buffer(tokens, d.q_heads, d.head_dim), buffer(tokens, d.q_heads, d.head_dim)
        self.projected, self.mlp_out = buffer(tokens, d.width), buffer(tokens, d.width)
        H, K = d.q_heads, d.kv_heads
        q, k, v = self.qkv[:, :H], self.qkv[:, H:H + K], self.qkv[:, H + K:]
        # the first norm has no block before it: its input is the embedding alone
        self.first = decode.BlockNorm(self.hidden, self.hidden, None, self.normed, d.layers[0]["attention_norm"],
                                      residual_scale=0.0)
        self.calls = []
        workspace = None
        for i, w in enumerate(d.layers):
            follows = d.layers[i + 1]["attention_norm"] if i + 1 < len(d.layers) else d.last_norm
            attention = decode.PagedAttention(self.rotated, w["cache"], d.page_table, self.q_start, self.context, self.attended,
                                              max_new=max_new, max_context=d.max_context, window=d.window, sinks=d.sinks,
                                              status=self.status, workspace=workspace)
            workspace = attention.workspace     # one for all layers: they follow one another
            self.calls.append(dict(
                append=decode.AppendKV(q, k, v, d.cos, d.sin, w["cache"], d.page_table, self.q_start, self.context,
                                       self.rotated, status=self.status),
                attention=attention,
                before_mlp=decode.BlockNorm(self.projected, self.hidden, self.hidden, self.normed, w["mlp_norm"]),
                after_mlp=decode.BlockNorm(self.mlp_out, self.hidden, self.hidden, self.normed, follows,
                                           post_weight=w["after_mlp"], gate=w["gate"])))
        self.logits = buffer(d.sequences, d.vocab)
        self.uniform = buffer(d.sequences, dtype=torch.float32)
        self.next = buffer(d.sequences, dtype=torch.int32)
        self.temperature, self.top_p = buffer(d.sequences, dtype=torch.float32), buffer(d.sequences, dtype=torch.float32)
        self.sampler = decode.Sampler(self.logits, self.uniform, self.next, temperature=self.temperature, top_p=self.top_p)

    def _mlp(self, weights):
        """The resident sparse layer over all tokens, up to four a launch."""
        d, lib, stream = self.decoder, _native.library(), torch.cuda.current_stream().cuda_stream
        for t in range(0, self.tokens, 4):
            rc = lib.ls_hip_core_layer_noalloc(d.width, 64, min(4, self.tokens - t), weights["mlp"].data_ptr(), d.groups,
                                               weights["mlp_scales"].data_ptr(), d.groups, d.core.data_ptr(), d.core_count,
                                               self.normed[t].data_ptr(), self.mlp_out[t].data_ptr(), None, None, stream)
            if rc:
                raise RuntimeError(f"Native core_layer_noalloc failed: {rc}")

    def run(self, ids, lengths, uniform, temperature=0.0, top_p=1.0):
        """ids: the sequences' new tokens one after another; lengths: (new tokens, context with them) of each.
        Returns the drawn token of every sequence (int32, on the GPU); that of one without new tokens means nothing."""
        d = self.decoder
        if len(lengths) != d.sequences or ids.numel() != self.tokens or sum(n for n, _ in lengths) != self.tokens:
            raise ValueError(f"the step is bound to {self.tokens} tokens of {d.sequences} sequences")
        if not all(0 <= n <= min(k, self.max_new) and k <= d.max_context for n, k in lengths):
            raise ValueError(f"a sequence of this step has up to {self.max_new} new tokens and {d.max_context} with them")
        ends = np.cumsum([0] + [n for n, _ in lengths])
        self.q_start.copy_(torch.from_numpy(ends.astype(np.int32)))
        self.context.copy_(torch.tensor([k for _, k in lengths], dtype=torch.int32))
        self.uniform.copy_(uniform)
        self.temperature.fill_(temperature)
        self.top_p.fill_(top_p)
        torch.index_select(d.embedding, 0, ids, out=self.hidden)
        self.first.enqueue()
        for w, c in zip(d.layers, self.calls):
            torch.mm(self.normed, w["qkv"], out=self.qkv.view(self.tokens, -1))
            c["append"].enqueue()
            c["attention"].enqueue()
            torch.mm(self.attended.view(self.tokens, -1), w["out"], out=self.projected)
            c["before_mlp"].enqueue()
            self._mlp(w)
            c["after_mlp"].enqueue()
        last = torch.from_numpy(np.maximum(ends[1:] - 1, 0)).to(DEV)
        torch.mm(self.normed[last], d.head, out=self.logits)
        self.sampler.enqueue()
        return self.next


def main():
    decoder = Decoder(window=128, sinks=4)
    prompts = [37, 5, 64, 18]
    g = torch.Generator(device=DEV).manual_seed(7)
    ids = torch.randint(0, decoder.vocab, (sum(prompts),), device=DEV, generator=g)
    drawn = decoder.bind(sum(prompts), max(prompts)).run(ids, [(n, n) for n in prompts], torch.rand(4, device=DEV, generator=g),
                                                        temperature=0.8, top_p=0.9)
    out = [drawn.tolist()]
    step = decoder.bind(4, 1)
    for i in range(1, 16):
        drawn = step.run(drawn, [(1, n + i) for n in prompts], torch.rand(4, device=DEV, generator=g), temperature=0.8, top_p=0.9)
        out.append(drawn.tolist())
    for s, row in enumerate(zip(*out)):
        print(f"sequence {s}: {prompts[s]} prompt tokens, then", *row)
    assert int(step.status) == 0


if __name__ == "__main__":
    main()
