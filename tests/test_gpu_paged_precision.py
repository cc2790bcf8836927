"""How exact paged attention is over fp16 pages: its error is that of rounding
the exact result to fp16."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import paged_util as pu
from test_gpu_paged import i32, randh

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hq,hkv,d,lengths", [
    (14, 2, 64, [2, 33, 300, 1001]),   # Qwen2.5-0.5B heads
    (32, 32, 128, [5, 64, 700]),       # Llama-2-7B heads
    (32, 2, 64, [100, 1500]),          # two tiles of heads
    (14, 2, 64, [40001]),              # parts
    (8, 8, 64, [60] * 300),            # one warp per CTA
])
@pytest.mark.parametrize("scale", [0.1, 1.5, 8.0])
def test_error_is_that_of_the_last_rounding(cuda, ops, hq, hkv, d, lengths, scale):
    """Root mean squares over each token's outputs. Beside the last rounding
    there are the scores' errors (a few 2^-24 of at most 2^6), the powers' (2^-21)
    and the sums', which enter squared: less than a thousandth of the rounding's
    2^-12. The rounding's own share differs where the computed value falls on the
    other side of a rounding border, so 1.02 is allowed; probabilities rounded to
    fp16 as well would give up to 1.4."""
    rng = np.random.default_rng(hq + d + len(lengths))
    table, n_pages = pu.page_table(rng, lengths, 16)
    cache, k, v = pu.random_cache(rng, ops, torch.float16, n_pages, hkv, 16, d, table)
    q = randh(rng, len(lengths), hq, d, scale=scale)
    got = ops.attention_paged(q.cuda(), cache, i32([n - 1 for n in lengths]), i32(range(len(lengths)))).cpu().double()
    want = torch.stack([pu.attention(q[t].double(), pu.rows_of(k, table, t, n), pu.rows_of(v, table, t, n))[0]
                        for t, n in enumerate(lengths)])
    off, least = (got - want).square().mean((1, 2)).sqrt(), (want.half().double() - want).square().mean((1, 2)).sqrt()
    assert (off <= 1.02 * least).all(), (off / least)[:8]


@pytest.mark.parametrize("dims,lengths", [((64, 2), [1, 2, 40, 1001, 30000]), ((128, 4), [1, 33, 700]),
                                          ((64, 8), [60] * 300)])
def test_infinite_values_stay_infinite(cuda, ops, dims, lengths):
    """A value that overflowed fp16 gives its infinity in its own dimension,
    infinities of both signs NaN, and nothing elsewhere; at a position whose
    power is the largest (exact in fp16) and at others."""
    rng = np.random.default_rng(len(lengths))
    d, hkv = dims
    hq = 4 * hkv
    table, n_pages = pu.page_table(rng, lengths, 16)
    cache, k, v = pu.random_cache(rng, ops, torch.float16, n_pages, hkv, 16, d, table)
    q = randh(rng, len(lengths), hq, d, scale=0.5)
    q[::2] = 0.0  # equal powers
    inf = float("inf")
    for t, n in enumerate(lengths):
        for at, dim, value in ((0, 3, inf), (n // 2, 9, -inf), (n - 1, 20, inf), (n - 1, 3, inf), (n // 3, 40, inf),
                               (n // 4, 40, -inf if n > 11 else inf), (n - 1, d - 1, float("nan"))):
            page, row = int(table[t, at // 16]), at % 16
            cache.v_pages[page, :, row, dim] = value
            v[page, :, row, dim] = value
    got = ops.attention_paged(q.cuda(), cache, i32([n - 1 for n in lengths]), i32(range(len(lengths)))).cpu().double()
    special = [3, 9, 20, 40, d - 1]
    rest = [i for i in range(d) if i not in special]
    for t, n in enumerate(lengths):
        want, _ = pu.attention(q[t].double(), pu.rows_of(k, table, t, n), pu.rows_of(v, table, t, n))
        assert torch.equal(got[t][:, special].nan_to_num(nan=7.0), want[:, special].nan_to_num(nan=7.0)), n
        assert torch.isfinite(got[t][:, rest]).all()
        # half a step of fp16 below 8 is 2^-9; the probabilities' 2^-21 and the sums' roundings are far below the rest
        assert float(want[:, rest].abs().max()) < 8 and ((got[t] - want)[:, rest].abs() <= 2e-3).all()
