"""The paged cache at its edges: rows of the table that end inside a tile, pools that run out, tokens without a place, and callers that want to see what is computed."""
import random

import pytest
import torch

import gpuk_b200 as gpuk
from tests.test_paged_gpu import BF16, F16, _Batch, _ints, _status_ok

pytestmark = pytest.mark.gpu


# ---- tables that end inside a tile ---------------------------------------------------------------------------
def _cut(ctx, new, heads, kv, hd, page, width, dtype=BF16, **more):
    """A batch whose table has fewer pages than some requests' tokens: what a token sees ends with the row."""
    b = _Batch(ctx, new, heads, kv, hd, page, dtype, **more)
    room, full = width * page, b.seen
    b.tables = b.tables[:, :width]
    b.keys, b.values = [k[:room] for k in b.keys], [v[:room] for v in b.values]
    b.seen = lambda i: full(i)[:, :room]
    return b


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("heads,kv,hd,page,width,ctx,new,dtype", [(8, 1, 128, 16, 2, [16], [64], BF16), (64, 8, 128, 16, 5, [0, 3], [200, 2], BF16), (8, 1, 64, 8, 1, [0], [40], F16),
                                                                 (64, 8, 64, 32, 3, [90, 96, 7], [150, 33, 60], F16), (128, 1, 128, 8, 9, [70], [9], BF16), (5, 5, 64, 8, 17, [0], [250], BF16),
                                                                 (16, 2, 128, 64, 1, [0, 64], [70, 20], BF16)])
def test_tiles_behind_the_table_s_end(heads, kv, hd, page, width, ctx, new, dtype, masked):
    """Tiles that begin behind the last key of the row: keys that are not there weigh nothing, whichever kernel takes the call."""
    b = _cut(ctx, new, heads, kv, hd, page, width, dtype, seed=heads + page, words=8 if masked else None)
    got = b.run()
    b.check(got)
    if not masked:
        b.check(b.run(max_new=1))
