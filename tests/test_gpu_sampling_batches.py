"""The same row alone and in calls of other numbers of rows (decode.Sampler), with random numbers and top-p at the edges
between two tokens, within the tolerance of test_gpu_sampling: either token of an edge is right, and which one may
depend on the number of rows, as the sums of a row without top-k are rounded chunk by chunk.
"""
import pytest

from test_gpu_sampling import accepted, log, random_rows, ranked, run

pytestmark = pytest.mark.gpu


def near(torch, x):
    """fp32 numbers around x."""
    x = torch.tensor(x, dtype=torch.float32)
    return [float(torch.nextafter(x, torch.tensor(0.0))), float(x), float(torch.nextafter(x, torch.tensor(1.0)))]


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("vocab", [9000, 60001])
@pytest.mark.parametrize("filters", ["none", "top_p", "top_p and min_p", "top_k and top_p"])
def test_edges_alone_and_in_batches(torch_gpu, vocab, dtype, filters):
    torch = torch_gpu
    logits, _, g = random_rows(torch, 1, vocab, dtype, vocab + 7, peaks=1, spread=1.0)
    row = logits[0].cpu()
    order, w = ranked(torch, row, 1.0)
    k = 900 if "top_k" in filters else 0
    ranks = w[order][: k or None]
    share = torch.cumsum(ranks, 0) / ranks.sum()
    settings = []
    for cut in (0.35, 0.8, 0.97):
        edge = int((share < cut).sum())
        for p in near(torch, float(share[edge])) if "top_p" in filters else [1.0]:
            kept = order[: k or None][: edge + 1] if "top_p" in filters else order[: k or None]
            # between two tokens' weights: of tokens at min_p itself the helper expects all to stay
            m = float((ranks[edge // 2] + ranks[ranks < ranks[edge // 2]][0]) / 2) if "min_p" in filters else 0.0
            ids = kept[w[kept] >= m].sort()[0]
            upto = torch.cumsum(w[ids], 0) / w[ids].sum()
            for at in (0.1, 0.5, 0.9):
                settings += [(p, m, u) for u in near(torch, float(upto[int(at * len(ids))]))]
    log("case:", vocab, dtype, filters, len(settings))
    ok = [accepted(torch, row, 1.0, k, p, m, u) for p, m, u in settings]
    for rows in (1, 3, 300):
        for i in range(0, len(settings), rows):
            some = (settings[i: i + rows] * rows)[:rows]
            tokens, logs = run(torch, row.cuda()[None].expand(rows, vocab).contiguous(), [u for _, _, u in some], None,
                               [k] * rows, [p for p, _, _ in some], [m for _, m, _ in some])
            for r in range(min(rows, len(settings) - i)):
                wants = ok[i + r].get(tokens[r])
                assert wants, (rows, settings[i + r], tokens[r], ok[i + r])
                assert any(abs(logs[r] - x) <= 1e-5 + 1e-6 * abs(x) for x in wants), (rows, settings[i + r])
