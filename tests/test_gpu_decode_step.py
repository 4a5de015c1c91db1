"""The operators together, as a decoder uses them (leanstream_amd.decode_step): prompts in one chunk, in pieces
and token by token fill the caches alike and lead to the same next tokens.

Between a chunk (tiles of many rows) and single tokens (few rows) the fp16 roundings of attention differ by
2^-11 of the values; hidden states are of order 1 to 4 and pass two layers, so the logits (order 1) may differ by a
few hundredths. Caches are compared with the same bound. Greedy tokens are compared where the best logit
leads by more than that.
"""
import pytest

pytestmark = pytest.mark.gpu

BOUND = 0.06


def fill(torch, decoder, prompts, ids, pieces):
    """Feeds the prompts in `pieces` tokens a time (the first piece takes the remainder); returns the last logits."""
    ends = [0]
    for n in prompts:
        ends.append(ends[-1] + n)
    done = [0] * len(prompts)
    u = torch.full((len(prompts),), 0.5, device="cuda")
    while any(d < n for d, n in zip(done, prompts)):
        left = max(n - d for d, n in zip(done, prompts))
        # sequences finish together: the longer ones go first, the others idle
        new = [max(0, min(pieces, n - d)) if n - d > left - pieces else 0 for d, n in zip(done, prompts)]
        take = torch.cat([ids[ends[s] + done[s]: ends[s] + done[s] + new[s]] for s in range(len(prompts))])
        done = [d + m for d, m in zip(done, new)]
        step = decoder.bind(sum(new), max(new))
        step.run(take, list(zip(new, done)), u)
        torch.cuda.synchronize()
        assert int(step.status) == 0
    return step.logits.float().clone(), step.next.clone()


@pytest.mark.parametrize("window,sinks", [(0, 0), (24, 4)])
def test_prompts_in_pieces(torch_gpu, window, sinks):
    torch = torch_gpu
    from leanstream_amd.decode_step import Decoder

    prompts = [61, 61, 61, 61]
    g = torch.Generator(device="cuda").manual_seed(3)
    ids = torch.randint(0, 2048, (sum(prompts),), device="cuda", generator=g)
    seen = []
    for pieces in (61, 20, 1):
        decoder = Decoder(window=window, sinks=sinks, max_context=64)
        for w in decoder.layers:
            w["cache"].k.zero_()
            w["cache"].v.zero_()
        logits, tokens = fill(torch, decoder, prompts, ids, pieces)
        assert logits.isfinite().all()
        seen.append((logits, tokens, [w["cache"].k.float() for w in decoder.layers], [w["cache"].v.float() for w in decoder.layers]))
    for logits, tokens, k, v in seen[1:]:
        assert (logits - seen[0][0]).abs().max() < BOUND
        top = seen[0][0].topk(2, dim=1)[0]
        clear = top[:, 0] - top[:, 1] > 2 * BOUND
        assert torch.equal(tokens[clear], seen[0][1][clear])
        for a, b in zip(k + v, seen[0][2] + seen[0][3]):
            assert (a - b).abs().max() < BOUND


def test_the_example_runs(torch_gpu, capsys):
    from leanstream_amd import decode_step

    decode_step.main()
    first = capsys.readouterr().out
    assert first.count("sequence") == 4
    decode_step.main()
    assert capsys.readouterr().out == first     # equal random numbers draw equal tokens
