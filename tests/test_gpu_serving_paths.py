"""Attention over the cache by every path that its sizes choose (test_serving_paths.py
pins which): tiles of 16 and 128 rows, some whole and the others in shares of
their keys, against the definition in 64 bits."""
import numpy as np
import pytest
import torch

from gpu_util import gen, normal
from test_gpu_serving import check_attention, filled, ints
from test_serving_paths import PATHS, rows_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", PATHS)
def test_attention_by_path(pkg, dev, name):
    path = PATHS[name][0]
    rows, requests, heads, kv_heads, d, block, width, bf16 = path
    dtype = torch.bfloat16 if bf16 else torch.float16
    n, blocks = rows_of(path), 2 * width
    cache, (k, v) = filled(pkg, dev, blocks, kv_heads, d, block, 117)
    g = gen(118)
    table = torch.randint(0, blocks, (requests, width), generator=g, dtype=torch.int32).to(dev)
    lens = [min(width * block, max(m, width * block - int(torch.randint(0, 300, (1,), generator=g)))) for m in n]
    cu = [0] + np.cumsum(n).tolist()
    q = normal((cu[-1], heads, d), 119, 1.5, dtype=dtype).to(dev)
    call = lambda: pkg.kv_attention(q, cache, table, ints(dev, *lens), cu=ints(dev, *cu) if rows else None)  # noqa: E731
    got = call()
    # rows of the first, the last and some tiles between, each as a request of its own
    at = sorted({*range(3), *range(cu[-1] - 3, cu[-1]), *np.linspace(0, cu[-1] - 1, 9).astype(int).tolist()})
    for t in at:
        r = int(np.searchsorted(cu, t, side="right")) - 1
        seen = lens[r] - n[r] + (t - cu[r]) + 1
        check_attention(got[t:t + 1], q[t:t + 1], k, v, block, table[r:r + 1], ints(dev, seen), [0, 1], d ** -0.5, blocks,
                        (name, t))
    assert all(torch.equal(call(), got) for _ in range(3))  # (whichever share arrives last)
