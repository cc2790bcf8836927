"""int8 rows of the paged append against the plain fp32 quotients, bit for bit:
scale = max|x| / 127 and code = x / scale rounded to nearest even. The values
reach the quantisation exactly (no norm, position 0 or value rows)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from test_gpu_paged import i32

pytestmark = pytest.mark.gpu


def plain(x):
    """Codes and scales of fp32 rows by IEEE division."""
    scale = x.abs().amax(-1) / 127
    return torch.round(x / scale[..., None]).to(torch.int8), scale


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("exponent", [-14, 0, 14])
def test_every_pair_of_fp16_values(cuda, ops, d, exponent):
    """All significands of the largest value against all of the values up to
    nine powers of two below it (smaller ones have code 0)."""
    most = torch.arange(1024, 2048, dtype=torch.float64) / 1024 * 2.0 ** exponent
    x = (torch.arange(1024, 2048, dtype=torch.float64)[None] / 1024
         * 2.0 ** torch.arange(exponent, exponent - 9, -1, dtype=torch.float64)[:, None]).flatten()
    x = x.half().float().unique()  # subnormals lose some bits: what is left of them
    x = torch.cat([x, torch.zeros(-len(x) % (d - 1))]).view(-1, d - 1)  # one row per token, beside the largest value
    tokens, hkv = len(x), len(most)
    rows = torch.cat([most.float().view(1, hkv, 1).expand(tokens, -1, -1), x[:, None].expand(-1, hkv, -1)], -1)
    rows = torch.where(rows.abs() > most.float().view(1, hkv, 1), 0.0, rows)
    rows[:, :, 2::3] *= -1
    v = rows.half().cuda()
    assert torch.equal(v.float().cpu(), rows)
    cache = ops.PagedKVCache.allocate(1, 256, hkv, d, 1, 1, dtype=torch.int8)
    cache.page_table.zero_()
    assert tokens <= 256
    ops.qkv_norm_rope_kv_append_paged(v[:, :1].clone(), v, v, cache, i32(np.arange(tokens)), i32(np.zeros(tokens)), 1e4)
    codes, scales = plain(rows)
    assert torch.equal(cache.v_scales[0, :, :tokens].cpu().T, scales)
    assert torch.equal(cache.v_pages[0, :, :tokens].cpu().transpose(0, 1), codes)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("near_half", [False, True])
def test_fp32_values(cuda, ops, d, near_half):
    """Values that come as fp32 biases: random ones, and ones next to the
    quotients half way between two codes, where the last bit decides."""
    rng = np.random.default_rng(d)
    hkv = 4096
    cache = ops.PagedKVCache.allocate(1, 8, hkv, d, 1, 1, dtype=torch.int8)
    cache.page_table.zero_()
    zero = torch.zeros(1, hkv, d, dtype=torch.float16, device="cuda")
    for i in range(4):
        most = torch.from_numpy(rng.uniform(1, 2, hkv) * 2.0 ** rng.integers(-58, 60, hkv)).float()
        if near_half:
            half = torch.from_numpy(rng.integers(-127, 127, (hkv, d)) + 0.5)
            x = (half * (most / 127).double()[:, None]).float()
            x = (x.view(torch.int32) + torch.from_numpy(rng.integers(-2, 3, (hkv, d))).int()).view(torch.float32)
        else:
            x = (torch.from_numpy(rng.uniform(-1, 1, (hkv, d))) * most[:, None]).float()
        x[:, 5] = most
        assert bool((x.abs() <= most[:, None]).all())
        bias = x.flatten().cuda()
        ops.qkv_norm_rope_kv_append_paged(zero[:, :1].clone(), zero, zero, cache, i32([0]), i32([0]), 1e4, bk=bias,
                                          bv=bias)
        codes, scales = plain(x)
        for got, got_scale in ((cache.k_pages, cache.k_scales), (cache.v_pages, cache.v_scales)):
            assert torch.equal(got_scale[0, :, 0].cpu(), scales)
            off = got[0, :, 0].cpu() != codes
            assert not off.any(), (x[off][:4], scales[off.any(1)][:4], got[0, :, 0].cpu()[off][:4], codes[off][:4])
