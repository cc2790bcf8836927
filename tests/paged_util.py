"""Plain forms of the paged-cache operators in 64 bits, and error bounds that
follow from the kernels' roundings (no test functions here).

Everything is computed by torch on the CPU in float64 from the same fp16 /
int8 / fp32 inputs. E16 and E32 are half a step of fp16 and fp32 relative to
the value."""
from __future__ import annotations

import math

import numpy as np
import torch

E16 = torch.finfo(torch.float16).eps / 2   # 2^-11
E32 = torch.finfo(torch.float32).eps / 2   # 2^-24
TINY16 = 2.0 ** -25                        # half a step of fp16's subnormals


def page_table(rng, lengths, page, n_spare=3, min_pages=1):
    """Random page table [n_seqs, max_pages] for sequences of these lengths and
    the number of pages; unused entries hold an id far out of range."""
    need = [-(-int(n) // page) for n in lengths]
    ids = rng.permutation(sum(need) + n_spare).astype(np.int32)
    table = np.full((len(need), max([min_pages, *need])), 1 << 30, np.int32)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = ids[at:at + n]
        at += n
    return table, sum(need) + n_spare


def quantise(x):
    """Codes and fp32 scales of float64 rows, as the append defines them."""
    amax = x.abs().amax(-1)
    scale = (amax / 127).float()
    code = torch.where(amax[..., None] > 0, torch.round(x * (127 / amax.clamp(min=1e-300))[..., None]), 0.0)
    return code.to(torch.int8), scale


def random_cache(rng, ops, dtype, n_pages, hkv, page, d, table, device="cuda:0", scale=1.0):
    """A PagedKVCache of normal rows on the device, and its dense float64 rows
    k, v [n_pages, hkv, page, d] on the CPU."""
    dense, parts = [], []
    for _ in range(2):
        x = torch.from_numpy(rng.standard_normal((n_pages, hkv, page, d)) * scale)
        if dtype == torch.int8:
            code, s = quantise(x)
            dense.append(code.double() * s.double()[..., None])
            parts.append((code.to(device), s.to(device)))
        else:
            h = x.half()
            dense.append(h.double())
            parts.append((h.to(device), None))
    cache = ops.PagedKVCache(parts[0][0], parts[1][0], torch.from_numpy(table).to(device), parts[0][1], parts[1][1])
    return cache, dense[0], dense[1]


def rows_of(dense, table, seq, n):
    """The first n rows of a sequence, [hkv, n, d]."""
    page = dense.shape[2]
    ids = torch.from_numpy(table[seq, :-(-n // page)].astype(np.int64))
    return dense[ids].permute(1, 0, 2, 3).flatten(1, 2)[:, :n]


def attention(q, k, v):
    """One token: q [hq, d], k and v [hkv, n, d], float64. Returns the output
    [hq, d] and a bound on the kernel's error.

    The kernel's errors: scores from exact fp16 / code products summed in fp32
    (at most d + 4 roundings, the tensor core's accumulation counted as two
    each), int8 with a query off by 2^-21 of its head's largest value, move an
    exponent by delta; a probability is then rounded to fp16
    (E16, and an absolute 2^-25 against a largest of at least 2^11, times the
    ratio of value scales for int8, for the ones below fp16's normal range);
    sums over n positions add 2 n E32 relative to sum p |v|, the quotient and
    its rounding to fp16 E16 relative to the result."""
    hq, d = q.shape
    g = hq // k.shape[0]
    n = k.shape[1]
    kk, vv = k.repeat_interleave(g, 0), v.repeat_interleave(g, 0)
    s = torch.einsum("hd,hjd->hj", q, kk) / math.sqrt(d)
    p = torch.softmax(s, -1)
    o = torch.einsum("hj,hjd->hd", p, vv)
    size = torch.einsum("hd,hjd->hj", q.abs(), kk.abs()) / math.sqrt(d)
    digits = 2.0 ** -21 * q.abs().amax(-1) * kk.abs().sum(-1).amax(-1) / math.sqrt(d)
    delta = (2 * (d + 8) * E32 * size.amax(-1) + digits + 8 * E32 * (s.abs().amax(-1) + 16) + 4 * E32)[:, None]
    spread = torch.einsum("hj,hjd->hd", p, vv.abs())
    vmax = vv.abs().amax((1, 2))[:, None]
    bound = (E16 + 2 * delta + 4 * n * E32) * (spread + o.abs()) + n * 2.0 ** -28 * vmax + E16 * o.abs() + TINY16
    return o, bound


def norm_rope(q, k, v, bq, bk, bv, qn, kn, eps, theta, positions):
    """float64 q, k, v after bias, norm and rotation, and per head the largest
    magnitude that entered the rotation (the scale of its rounding errors)."""
    d = q.shape[2]
    out, sizes = [], []
    freq = float(theta) ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
    angle = torch.as_tensor(positions, dtype=torch.float64)[:, None] * freq
    c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    for x, b, w, turn in ((q, bq, qn, True), (k, bk, kn, True), (v, bv, None, False)):
        x = x.double()
        if b is not None:
            x = x + b.double().view(1, -1, d)
        if w is not None:
            x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()
        sizes.append(x.abs().amax(-1, keepdim=True))
        if turn:
            a, e = x[..., :d // 2], x[..., d // 2:]
            x = torch.cat([a * c - e * s, e * c + a * s], -1)
        out.append(x)
    return out, sizes


# fp32 errors of bias, norm, sine and rotation relative to the largest value of
# the head: bias 1, norm at most d + 8 halves of which the sum's d enter as
# their square root's half, weight 2, sine 4 and rotation 3 roundings; 96 of
# them bound every head_dim
ROPE_ERR = 96 * E32


def f16_bound(want, size):
    return E16 * want.abs() + ROPE_ERR * size + TINY16
