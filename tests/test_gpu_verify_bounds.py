"""verify with bounds that do not ascend: every row belongs to one request at
most, and nothing of an earlier call decides."""
import random

import pytest
import torch

from gpu_util import gen

pytestmark = pytest.mark.gpu


def ranges(cu, rows):
    """The rows of each request: bounds count as the nearest ones in order."""
    out = []
    for a, b in zip(cu, cu[1:]):
        first = min(max(a, 0), rows)
        out.append((first, min(max(b, first), rows)))
    return out


def owner(cu, row, rows):
    """The request that a row is judged for: the one that a search for it ends at."""
    lo, hi = 0, len(cu) - 1
    while hi - lo > 1:
        mid = (lo + hi) // 2
        lo, hi = (mid, hi) if cu[mid] <= row else (lo, mid)
    first, end = ranges(cu, rows)[lo]
    return lo if first <= row < end else -1


@pytest.mark.parametrize("certain", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_bounds_that_do_not_ascend(pkg, dev, dtype, certain):
    V, T = 3000, 12
    g = gen(3)
    x = (torch.randn((T, V), generator=g) * 2).to(dtype)
    q = (x.double() + 0.4 * torch.randn((T, V), generator=g, dtype=torch.float64)).softmax(-1)
    drafts = torch.multinomial(q, 1, generator=g)[:, 0]
    u = torch.rand(T, generator=g) * (0.05 if certain else 0.8)
    x, q, drafts, u = x.to(dev), q.float().to(dev), drafts.to(dev), u.to(dev)
    # what an earlier call leaves: every row but the requests' last accepted, with thresholds that keep everything
    best = x.double().argmax(-1)
    under = (x.double().softmax(-1) * (1 - 1e-6)).float()

    def earlier():
        got = pkg.verify(x, best, torch.zeros_like(u), torch.zeros(6, device=dev),
                         cu=torch.tensor([0, 12, 12, 12, 12, 12, 12], dtype=torch.int32, device=dev), draft_probs=under)
        assert got.counts.tolist() == [12, 0, 0, 0, 0, 0]

    rng = random.Random(5)
    bounds = [[0, 5, 0, 0, 0], [0, 6, 2, 4, 5], [0, 12, 0, 12], [12, 0], [4, 0, 12], [0, 3, 1, 2, 12], [-4, 7, 3, 99, 5, 12]]
    bounds += [[rng.randint(-2, T + 2) for _ in range(rng.randint(2, 7))] for _ in range(25)]
    for cu in bounds:
        R = len(cu) - 1
        draw = torch.rand(R, generator=g).to(dev)
        probs = None if certain else q
        owners, tokens, counts = [owner(cu, i, T) for i in range(T)], [-1] * T, []
        for r, (a, b) in enumerate(ranges(cu, T)):
            if a == b:
                counts.append(0)
                continue
            alone = pkg.verify(x[a:b], drafts[a:b], u[a:b], draw[r:r + 1], cu=torch.tensor([0, b - a], dtype=torch.int32, device=dev),
                               draft_probs=None if certain else q[a:b], top_p=0.9)
            n = int(alone.counts[0])
            stop = min([a + n - 1] + [i for i in range(a, b) if owners[i] != r])
            for i in range(a, stop + 1):
                if owners[i] == r:
                    tokens[i] = int(alone.tokens[i - a])
            counts.append(stop - a + 1)
        for _ in range(2):
            earlier()
            got = pkg.verify(x, drafts, u, draw, cu=torch.tensor(cu, dtype=torch.int32, device=dev), draft_probs=probs, top_p=0.9)
            assert got.tokens.tolist() == tokens and got.counts.tolist() == counts, cu


@pytest.mark.parametrize("with_cu", [False, True])
@pytest.mark.parametrize("with_probs", [False, True])
@pytest.mark.parametrize("requests", [1, 70, 3000])
def test_requests_without_rows_get_counts_of_zero(pkg, dev, requests, with_probs, with_cu):
    """The C entry with no rows at all: counts are written, with the draft's
    probabilities given (never read) or not."""
    counts = torch.full((requests + 1,), 7, dtype=torch.int32, device=dev)
    cu, draw = torch.zeros(requests + 1, dtype=torch.int32, device=dev), torch.zeros(requests, device=dev)
    probs = torch.zeros(8, device=dev)
    rc = pkg.load_library().hxmi_verify(0, None, None, None, draw.data_ptr(), cu.data_ptr() if with_cu else None,
                                        probs.data_ptr() if with_probs else None, 2, None, None, None, None, 1.0, 0, 1.0, 0.0,
                                        None, counts.data_ptr(), 0, requests, 1000, 1000, 1000, None, 0,
                                        torch.cuda.current_stream().cuda_stream)
    assert rc == 0, pkg.load_library().hxmi_last_error().decode()
    assert counts.tolist() == [0] * requests + [7]
