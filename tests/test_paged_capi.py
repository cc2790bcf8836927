"""Refusals of the paged-cache and log-probability entry points, on the CPU:
every bad argument is answered with its status before any GPU work."""
from __future__ import annotations

import ctypes

import pytest


@pytest.fixture(scope="module")
def capi():
    from littlellm_b200 import build
    build.build()
    from littlellm_b200 import _capi
    return _capi


P = 4096  # a 16-byte aligned address that is never dereferenced


def cache(capi, **kw):
    c = capi.PagedCache(P, P, P, P, P, 10, 16, 2, 64, 3, 4, capi.I8)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def append(capi, c, **kw):
    a = dict(q=P, qs=8 * 64, k=P, ks=128, v=P, vs=128, bq=None, bk=None, bv=None, bd=capi.F16, qn=None, kn=None,
             nd=capi.F16, eps=1e-6, theta=1e4, positions=P, seqs=P, n=4, heads=8, cache=c, out=P, os=8 * 64,
             err=None, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return capi.lib.kllm_b200_qkv_norm_rope_kv_append_paged(*a.values())


def read(capi, c, **kw):
    a = dict(cache=c, positions=P, seqs=P, n=4, slots=None, n_slots=0, max_seq=0, k=P, v=P, err=None, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return capi.lib.kllm_b200_kv_read_paged(*a.values())


def attend(capi, c, **kw):
    a = dict(q=P, qs=8 * 64, cache=c, positions=P, seqs=P, n=4, heads=8, out=P, os=8 * 64, ws=None, nbytes=0,
             err=None, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return capi.lib.kllm_b200_attention_paged(*a.values())


@pytest.mark.parametrize("call", [append, read, attend])
def test_cache_refusals(capi, call):
    for change, status in (
            (dict(cache_dtype=capi.F32), capi.ERR_DTYPE), (dict(cache_dtype=99), capi.ERR_DTYPE),
            (dict(head_dim=96), capi.ERR_SHAPE), (dict(head_dim=256), capi.ERR_SHAPE),
            (dict(page_size=4), capi.ERR_SHAPE), (dict(page_size=24), capi.ERR_SHAPE),
            (dict(page_size=0), capi.ERR_SHAPE), (dict(page_size=1 << 21), capi.ERR_SHAPE),
            (dict(n_pages=0), capi.ERR_SHAPE), (dict(n_kv_heads=0), capi.ERR_SHAPE), (dict(n_seqs=0), capi.ERR_SHAPE),
            (dict(max_pages=0), capi.ERR_SHAPE), (dict(n_pages=1 << 31), capi.ERR_SHAPE),
            (dict(n_kv_heads=65536), capi.ERR_SHAPE), (dict(max_pages=1 << 27), capi.ERR_SHAPE),
            (dict(n_pages=-1), capi.ERR_INVALID_ARG), (dict(n_seqs=-1), capi.ERR_INVALID_ARG),
            (dict(k_pages=None), capi.ERR_INVALID_ARG), (dict(v_pages=None), capi.ERR_INVALID_ARG),
            (dict(page_table=None), capi.ERR_INVALID_ARG), (dict(k_scales=None), capi.ERR_INVALID_ARG),
            (dict(v_scales=None), capi.ERR_INVALID_ARG), (dict(k_pages=P + 8), capi.ERR_ALIGN),
            (dict(v_pages=P + 2), capi.ERR_ALIGN)):
        assert call(capi, cache(capi, **change)) == status, change
        assert capi.last_error()
    assert call(capi, None) == capi.ERR_INVALID_ARG
    # no tokens: nothing to do, whatever the pointers
    none = dict(positions=None, seqs=None, n=0)
    assert call(capi, cache(capi), **none) == capi.OK
    assert call(capi, cache(capi), n=-1) == capi.ERR_INVALID_ARG
    assert call(capi, cache(capi), positions=None) == capi.ERR_INVALID_ARG
    assert call(capi, cache(capi), seqs=None) == capi.ERR_INVALID_ARG


def test_append_refusals(capi):
    c = cache(capi)
    for change, status in (
            (dict(q=None), capi.ERR_INVALID_ARG), (dict(k=None), capi.ERR_INVALID_ARG),
            (dict(v=None), capi.ERR_INVALID_ARG), (dict(out=None), capi.ERR_INVALID_ARG),
            (dict(q=P + 8), capi.ERR_ALIGN), (dict(out=P + 2), capi.ERR_ALIGN), (dict(bq=P + 4), capi.ERR_ALIGN),
            (dict(kn=P + 8), capi.ERR_ALIGN), (dict(qs=8 * 64 + 4, os=8 * 64 + 4), capi.ERR_ALIGN),
            (dict(ks=130), capi.ERR_ALIGN), (dict(qs=8 * 64 - 8), capi.ERR_SHAPE), (dict(os=0), capi.ERR_SHAPE),
            (dict(ks=64), capi.ERR_SHAPE), (dict(vs=-128), capi.ERR_SHAPE), (dict(os=8 * 64 + 8), capi.ERR_SHAPE),
            (dict(heads=0), capi.ERR_SHAPE), (dict(heads=-1), capi.ERR_INVALID_ARG),
            (dict(bq=P, bd=capi.I8), capi.ERR_DTYPE), (dict(qn=P, nd=capi.I32), capi.ERR_DTYPE),
            (dict(theta=0.0), capi.ERR_INVALID_ARG), (dict(theta=float("nan")), capi.ERR_INVALID_ARG),
            (dict(theta=float("inf")), capi.ERR_INVALID_ARG), (dict(eps=-1.0), capi.ERR_INVALID_ARG),
            (dict(eps=float("nan")), capi.ERR_INVALID_ARG)):
        assert append(capi, c, **change) == status, change


def test_read_refusals(capi):
    c = cache(capi)
    for change, status in (
            (dict(k=None), capi.ERR_INVALID_ARG), (dict(v=None), capi.ERR_INVALID_ARG), (dict(k=P + 8), capi.ERR_ALIGN),
            (dict(v=P + 2), capi.ERR_ALIGN), (dict(slots=P), capi.ERR_SHAPE),
            (dict(slots=P, n_slots=2), capi.ERR_SHAPE), (dict(slots=P, max_seq=2), capi.ERR_SHAPE),
            (dict(slots=P, n_slots=-2, max_seq=2), capi.ERR_INVALID_ARG)):
        assert read(capi, c, **change) == status, change


def test_attention_refusals(capi):
    c = cache(capi)
    for change, status in (
            (dict(q=None), capi.ERR_INVALID_ARG), (dict(out=None), capi.ERR_INVALID_ARG),
            (dict(heads=7), capi.ERR_SHAPE), (dict(heads=0), capi.ERR_SHAPE),
            (dict(heads=34, qs=34 * 64, os=34 * 64), capi.ERR_SHAPE), (dict(qs=8), capi.ERR_SHAPE),
            (dict(os=8 * 64 - 8), capi.ERR_SHAPE), (dict(qs=8 * 64 + 4), capi.ERR_ALIGN), (dict(q=P + 8), capi.ERR_ALIGN),
            (dict(out=P + 8), capi.ERR_ALIGN), (dict(nbytes=-1), capi.ERR_INVALID_ARG),
            (dict(nbytes=64), capi.ERR_ALIGN), (dict(ws=P + 4, nbytes=64), capi.ERR_ALIGN),
            (dict(n=1 << 31), capi.ERR_SHAPE)):
        assert attend(capi, c, **change) == status, change
    n = ctypes.c_int64(-1)
    size = capi.lib.kllm_b200_attention_paged_workspace_bytes
    assert size(4, 8, c, None) == capi.ERR_INVALID_ARG
    assert size(4, 8, None, n) == capi.ERR_INVALID_ARG and n.value == 0
    assert size(4, 7, c, n) == capi.ERR_SHAPE
    assert size(0, 8, c, n) == capi.OK and n.value == 0
    assert size(100_000, 8, c, n) == capi.OK and n.value == 0  # a batch that fills the device needs no parts


@pytest.mark.parametrize("n", [1 << 31, (1 << 57) + 1, (1 << 60) + 3, (1 << 63) - 1])
def test_counts_past_every_grid(capi, n):
    """Also those whose products with the kernels' tile counts pass 64 bits."""
    c = cache(capi)
    assert append(capi, c, n=n, out=4 * P) == capi.ERR_SHAPE
    assert read(capi, c, n=n) == capi.ERR_SHAPE
    assert attend(capi, c, n=n, out=4 * P) == capi.ERR_SHAPE
    assert capi.lib.kllm_b200_attention_paged_workspace_bytes(n, 8, c, ctypes.c_int64()) == capi.ERR_SHAPE
    assert capi.lib.kllm_b200_token_logprobs(P, capi.F16, n, 100, 100, P, P, P, P, 5, P, P, None, None) == capi.ERR_SHAPE


def test_more_items_than_a_grid_holds(capi):
    c = cache(capi, n_kv_heads=65535)
    wide = 65535 * 64
    assert attend(capi, c, n=1 << 20, heads=65535, qs=wide, os=wide, out=4 * P) == capi.ERR_SHAPE
    assert capi.lib.kllm_b200_attention_paged_workspace_bytes(1 << 20, 65535, c, ctypes.c_int64()) == capi.ERR_SHAPE


def test_attention_in_place_is_refused(capi):
    assert attend(capi, cache(capi)) == capi.ERR_INVALID_ARG


def test_logprob_refusals(capi):
    def call(**kw):
        a = dict(x=P, dtype=capi.F16, rows=2, vocab=100, stride=100, tokens=P, lp=P, ranks=P, h=P, k=5, ids=P, top=P,
                 err=None, stream=None)
        assert set(kw) <= set(a)
        a.update(kw)
        return capi.lib.kllm_b200_token_logprobs(*a.values())

    for change, status in (
            (dict(dtype=capi.I8), capi.ERR_DTYPE), (dict(rows=-1), capi.ERR_INVALID_ARG),
            (dict(vocab=0), capi.ERR_SHAPE), (dict(vocab=-1), capi.ERR_INVALID_ARG), (dict(stride=99), capi.ERR_SHAPE),
            (dict(vocab=1 << 31, stride=1 << 31), capi.ERR_SHAPE), (dict(rows=1 << 30), capi.ERR_SHAPE),
            (dict(k=33), capi.ERR_SHAPE), (dict(k=-1), capi.ERR_INVALID_ARG), (dict(vocab=4, k=5), capi.ERR_SHAPE),
            (dict(x=None), capi.ERR_INVALID_ARG), (dict(x=P + 1), capi.ERR_ALIGN),
            (dict(x=P + 2, dtype=capi.F32), capi.ERR_ALIGN), (dict(tokens=None), capi.ERR_INVALID_ARG),
            (dict(lp=None), capi.ERR_INVALID_ARG), (dict(ranks=None), capi.ERR_INVALID_ARG),
            (dict(ids=None), capi.ERR_INVALID_ARG), (dict(top=None), capi.ERR_INVALID_ARG)):
        assert call(**change) == status, change
    assert call(rows=0, x=None) == capi.OK


def test_wrappers_refuse_host_tensors_and_bad_shapes(capi):
    import torch

    from littlellm_b200 import ops
    pages = torch.zeros(4, 2, 16, 64, dtype=torch.float16)
    table = torch.zeros(1, 4, dtype=torch.int32)
    with pytest.raises(capi.KllmError) as e:
        ops.PagedKVCache(pages, pages, table)
    assert e.value.status == capi.ERR_INVALID_ARG
    with pytest.raises(capi.KllmError) as e:
        ops.token_logprobs(torch.zeros(2, 8))
    assert e.value.status == capi.ERR_INVALID_ARG
