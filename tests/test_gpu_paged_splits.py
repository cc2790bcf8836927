"""Paged attention over long caches, tile by tile: every tile of 32 positions
holds one position whose key a query asks for, together with an equal key in a
tile far away. The output is the mean of the two values, so a tile that is left
out or taken twice, or a part that joins with another weight, changes it by a
sixth of their difference at least, hundreds of times the bound, whatever the
sequence's length."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import paged_util as pu
from test_gpu_paged import DTYPES, flags, i32

pytestmark = pytest.mark.gpu

TILE = 32
HKV = 2


def paired_cache(ops, rng, dtype, n, d, page, capacity):
    """One sequence of n positions with keys of +-1, the pairs (position,
    position) that share a key, and the float64 values [HKV, n, d]."""
    tiles = -(-n // TILE)
    inside = rng.integers(0, TILE, tiles)
    inside[::3], inside[1::3] = 0, TILE - 1  # a tile's ends among them
    at = np.minimum(np.arange(tiles) * TILE + inside, n - 1)
    pairs = [(int(at[i]), int(at[tiles - 1 - i])) for i in range((tiles + 1) // 2)]
    keys = torch.from_numpy(rng.choice([-1.0, 1.0], (n, d)))
    for a, b in pairs:
        keys[b] = keys[a]
    table, n_pages = pu.page_table(rng, [n], page, min_pages=capacity // page)
    cache, _, v = pu.random_cache(rng, ops, dtype, n_pages, HKV, page, d, table)
    ids = torch.from_numpy(table[0, :-(-n // page)].astype(np.int64)).cuda()
    rows = torch.zeros(len(ids) * page, d)
    rows[:n] = keys
    rows = rows.view(len(ids), 1, page, d).expand(-1, HKV, -1, -1).cuda()
    if dtype == torch.int8:
        cache.k_pages[ids], cache.k_scales[ids] = (rows * 127).to(torch.int8), 1 / 127
    else:
        cache.k_pages[ids] = rows.half()
    # a query of 8 times a key scores sqrt(d) 8 with it; all others together weigh next to nothing
    for part in range(0, len(pairs), 256):
        some = pairs[part:part + 256]
        s = (keys[[a for a, _ in some]] @ keys.T) * (8 / d ** 0.5)
        for i, (a, b) in enumerate(some):
            s[i, [a, b]] = -np.inf
        assert float((s - 8 * d ** 0.5).exp().sum(1).max()) < 1e-6
    return cache, keys, pairs, pu.rows_of(v, table, 0, n)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,capacity,d,group,tokens,padded", [
    (65553, 65600, 64, 7, 1, 0),      # one token: clusters of eight, sixteen of them
    (40001, 65536, 128, 2, 1, 0),     # a sequence that fills part of the capacity
    (12345, 16384, 64, 9, 1, 0),      # two tiles of heads
    (700, 1024, 64, 7, 1, 0),         # one cluster
    (65553, 65600, 64, 7, 40, 20),    # more parts than run at once
    (20000, 65536, 128, 4, 5, 4),
    (9000, 9008, 64, 7, 400, 9),      # no parts; several waves, longest first
    (500, 512, 64, 7, 2000, 0),       # one warp per CTA
    (33, 512, 128, 1, 2000, 3),
])
def test_every_tile_counts_once(cuda, ops, dtype, n, capacity, d, group, tokens, padded):
    rng = np.random.default_rng(n + d)
    hq = group * HKV
    cache, keys, pairs, v = paired_cache(ops, rng, dtype, n, d, 8 if capacity % 16 else 16, capacity)
    positions = i32([n - 1] * tokens + [-1] * padded)
    seqs = i32([0] * tokens + [-1] * padded)
    todo = list(range(len(pairs)))
    asked = 0
    while asked < len(todo):
        which = np.resize(todo[asked:asked + tokens * hq], tokens * hq).reshape(tokens, hq)
        asked += tokens * hq
        q = torch.zeros(tokens + padded, hq, d, dtype=torch.float16)
        first, second = (torch.tensor([pairs[i][side] for i in which.ravel()]) for side in (0, 1))
        q[:tokens] = (8 * keys[first]).view(tokens, hq, d).half()
        err = flags()
        got = ops.attention_paged(q.cuda(), cache, positions, seqs, err_flags=err).cpu().double()
        assert int(err.item()) == 0 and bool((got[tokens:] == 0).all())
        head = torch.arange(hq).repeat(tokens) // group
        one, two = v[head, first], v[head, second]
        # the two probabilities are equal; E16 for their rounding and for the result's, the sums' roundings (two per
        # 16 positions, the tensor core's counted as two each), and what the other keys weigh
        bound = ((2 * pu.E16 + 4 * (n / 16 + 32) * pu.E32 + 4e-6) * (one.abs() + two.abs()) / 2 + 4e-6 * 8 + pu.TINY16)
        off = (got[:tokens].reshape(-1, d) - (one + two) / 2).abs() > bound
        assert not off.any(), [pairs[i] for i in which.ravel()[off.any(1).numpy()][:5]]
