"""Which tiles attention over the cache takes for a call: 16 or 128 rows, how
many of them run whole and in how many shares of their keys the others, from
the sizes alone.  PATHS are the calls that test_gpu_serving_paths.py runs."""
import pytest

# name: (rows of each request or None for one each, requests, query heads, kv heads, dim, block, width, bf16),
#       (rows of a tile, tiles that run whole, tiles in shares, shares)
PATHS = {
    "decode, some tiles shared": ((None, 280, 8, 2, 64, 64, 40, 0), (16, 512, 48, 10)),
    "decode of 128 dims, some tiles shared": ((None, 71, 32, 8, 128, 32, 70, 1), (16, 512, 56, 9)),
    "decode of 40 dims, whole rounds and one tile": ((None, 513, 5, 1, 40, 16, 200, 0), (16, 512, 1, 13)),
    "drafts, some tiles shared": (([1, 5, 2, 4, 3], 100, 21, 3, 64, 16, 60, 1), (16, 512, 181, 2)),
    "prompts of 128 dims, some tiles shared": (([9000, 0, 500], 3, 8, 2, 128, 64, 158, 0), (128, 512, 86, 5)),
    "prompts of 64 dims, some tiles shared": (([1500, 1601], 2, 24, 4, 64, 32, 120, 1), (128, 512, 76, 6)),
    "prompts of 80 dims, some tiles shared": (([4000, 3300], 2, 10, 1, 80, 256, 16, 1), (128, 512, 60, 8)),
    "a prompt, all tiles shared": (([347, 173], 2, 8, 2, 128, 32, 30, 0), (128, 0, 36, 2)),
    "a prompt of 64 dims, all tiles shared": (([433, 267], 2, 6, 1, 64, 32, 30, 1), (128, 0, 34, 2)),
}


def rows_of(path):
    rows, requests = path[:2]
    return [1] * requests if rows is None else (rows * requests)[:requests]


@pytest.mark.parametrize("name", PATHS)
def test_path(pkg, name):
    path, (tile, whole, shared, shares) = PATHS[name]
    rows, requests, heads, kv_heads, d, block, width, _ = path
    tokens, group = sum(rows_of(path)), heads // kv_heads
    tiles = tokens * group // tile + requests if rows else requests * -(-group // tile)
    assert tiles * kv_heads == whole + shared and shares > 1
    # a share's floats: 4 or 16 of O a lane for each 16 or 32 dims of 64 or 128, m, d and l
    part = (d // 64.1 + 1) * 16 + 3 if tile == 16 else 4 * ((d // 64.1 + 1) * 32 + 3)
    need = pkg.load_library().hxmi_kv_attention_workspace_bytes(tokens, requests, heads, kv_heads, d, block, width,
                                                                int(rows is not None))
    assert need == 16384 + shared * shares * int(part) * 256
