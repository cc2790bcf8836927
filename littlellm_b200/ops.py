"""torch-facing wrappers of the C ABI.

One function per operator of the reference interface
(``include/kllm/op/ops.h:10-35``: embedding, rms_norm, add_bias_inplace,
add_inplace, select_last_row, silu_mul, rope_inplace, copy_kv_to_cache,
dequantize_int8) plus the fused/batched entry points (add_rms_norm,
qkv_bias_rope_kv_append, select_last_rows, attention_head_major, linear,
linear_swiglu), the operators of a paged cache (PagedKVCache,
qkv_norm_rope_kv_append_paged, kv_read_paged, attention_paged) and
token_logprobs. Each takes CUDA tensors, passes
their device pointers to ``libkllm_b200.so`` on the tensor's current stream
and raises ``KllmError`` with the library's message on a non-zero status,
the way the reference throws ``std::runtime_error``.

torch supplies device memory and streams here; all arithmetic happens in the
library's kernels.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from . import _capi
from ._capi import F16, F32, I8, I32, KllmError, check, lib

try:  # without the Stream object and the lazy initialisation of the public functions: 1 us a call
    from torch._C import _cuda_getCurrentRawStream as _raw_stream, _cuda_getDevice as _current_device
except ImportError:  # names that torch does not promise
    def _raw_stream(index: int) -> int:
        return torch.cuda.current_stream(index).cuda_stream

    _current_device = torch.cuda.current_device

_DTYPES = {torch.float32: F32, torch.float16: F16, torch.int32: I32, torch.int8: I8}


def dtype_code(t: torch.Tensor) -> int:
    try:
        return _DTYPES[t.dtype]
    except KeyError:
        raise KllmError(_capi.ERR_DTYPE, f"unsupported tensor dtype {t.dtype}") from None


def _dev(*tensors):
    """Checks that every given tensor is a contiguous CUDA tensor on one device
    and returns that device."""
    device = None
    for t in tensors:
        if t is None:
            continue
        if not t.is_cuda:
            raise KllmError(_capi.ERR_INVALID_ARG, "expected a CUDA tensor")
        if not t.is_contiguous():
            raise KllmError(_capi.ERR_SHAPE, "expected a contiguous tensor")
        if device is None:
            device = t.device
        elif t.device != device:
            raise KllmError(_capi.ERR_INVALID_ARG, "tensors are on different devices")
    return device


def _ptr(t):
    return None if t is None else t.data_ptr()


def _stream(device) -> int:
    return _raw_stream(device.index)


def set_pdl(enable: bool) -> bool:
    """Launch mode of the individual entry points for this host thread
    (kllm_b200_set_pdl): programmatic dependent launch with the inputs no
    kernel of the library writes read before the dependency wait. Returns the
    previous mode."""
    return bool(lib.kllm_b200_set_pdl(1 if enable else 0))


def embedding(table: torch.Tensor, ids: torch.Tensor, out: torch.Tensor | None = None,
              err_flags: torch.Tensor | None = None) -> torch.Tensor:
    """out[t] = table[ids[t]] (reference embedding, ids on the device)."""
    if out is None:
        out = torch.empty((ids.numel(), table.shape[1]), dtype=table.dtype, device=table.device)
    dev = _dev(table, ids, out, err_flags)
    if ids.dtype != torch.int32:
        raise KllmError(_capi.ERR_DTYPE, "ids must be int32")
    with torch.cuda.device(dev):
        check(lib.kllm_b200_embedding(_ptr(table), table.shape[0], table.shape[1], dtype_code(table),
                                      _ptr(ids), ids.numel(), _ptr(out), dtype_code(out),
                                      _ptr(err_flags), _stream(dev)))
    return out


def embedding_host_ids(table: torch.Tensor, ids, out: torch.Tensor | None = None,
                       err_flags: torch.Tensor | None = None) -> torch.Tensor:
    """out[t] = table[ids[t]] with the ids in host memory (a sequence of ints,
    as the reference's cuda_embedding takes them); they travel in the kernel
    launches' parameters, no device buffer or blocking copy."""
    import numpy as np
    host = np.ascontiguousarray(np.asarray(ids, dtype=np.int32))
    if out is None:
        out = torch.empty((host.size, table.shape[1]), dtype=table.dtype, device=table.device)
    dev = _dev(table, out, err_flags)
    with torch.cuda.device(dev):
        check(lib.kllm_b200_embedding_host_ids(_ptr(table), table.shape[0], table.shape[1], dtype_code(table),
                                               host.ctypes.data, host.size, _ptr(out), dtype_code(out),
                                               _ptr(err_flags), _stream(dev)))
    return out


def embedding_rms_norm(table: torch.Tensor, ids: torch.Tensor, weight: torch.Tensor, eps: float,
                       residual: torch.Tensor | None = None, out: torch.Tensor | None = None,
                       err_flags: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """residual = table[ids] and out = rms_norm(residual) * weight, one launch
    (embedding + layer 0's input norm). Returns (residual, out)."""
    if ids.dtype != torch.int32:
        raise KllmError(_capi.ERR_DTYPE, "ids must be int32")
    if table.dtype != torch.float16:
        raise KllmError(_capi.ERR_DTYPE, "embedding_rms_norm takes an fp16 table")
    shape = (ids.numel(), table.shape[1])
    if residual is None:
        residual = torch.empty(shape, dtype=table.dtype, device=table.device)
    if out is None:
        out = torch.empty(shape, dtype=table.dtype, device=table.device)
    dev = _dev(table, ids, weight, residual, out, err_flags)
    with torch.cuda.device(dev):
        check(lib.kllm_b200_embedding_rms_norm(_ptr(table), table.shape[0], table.shape[1], _ptr(ids), ids.numel(),
                                               _ptr(weight), dtype_code(weight), eps, _ptr(residual), _ptr(out),
                                               _ptr(err_flags), _stream(dev)))
    return residual, out


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float,
             out: torch.Tensor | None = None) -> torch.Tensor:
    if out is None:
        out = torch.empty_like(x)
    dev = _dev(x, weight, out)
    hidden = x.shape[-1]
    with torch.cuda.device(dev):
        check(lib.kllm_b200_rms_norm(_ptr(x), _ptr(weight), _ptr(out), x.numel() // hidden, hidden,
                                     eps, dtype_code(x), dtype_code(weight), _stream(dev)))
    return out


def add_rms_norm(residual: torch.Tensor, delta: torch.Tensor | None, weight: torch.Tensor,
                 eps: float, out: torch.Tensor | None = None) -> torch.Tensor:
    """residual += delta (stored, fp16-rounded); returns RMSNorm(residual) * weight."""
    if out is None:
        out = torch.empty_like(residual)
    dev = _dev(residual, delta, weight, out)
    hidden = residual.shape[-1]
    with torch.cuda.device(dev):
        check(lib.kllm_b200_add_rms_norm(_ptr(residual), _ptr(delta), _ptr(weight), _ptr(out),
                                         residual.numel() // hidden, hidden, eps,
                                         dtype_code(residual), dtype_code(weight), _stream(dev)))
    return out


def add_inplace(x: torch.Tensor, y: torch.Tensor) -> torch.Tensor:
    dev = _dev(x, y)
    if x.numel() != y.numel():
        raise KllmError(_capi.ERR_SHAPE, "add shape mismatch")
    with torch.cuda.device(dev):
        check(lib.kllm_b200_add_inplace(_ptr(x), _ptr(y), x.numel(), dtype_code(x), dtype_code(y),
                                        _stream(dev)))
    return x


def add_bias_inplace(x: torch.Tensor, bias: torch.Tensor | None) -> torch.Tensor:
    if bias is None:
        return x
    dev = _dev(x, bias)
    cols = x.shape[-1]
    with torch.cuda.device(dev):
        check(lib.kllm_b200_add_bias_inplace(_ptr(x), _ptr(bias), x.numel() // cols, cols,
                                             dtype_code(x), dtype_code(bias), _stream(dev)))
    return x


def select_last_row(x: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    if out is None:
        out = torch.empty((1, x.shape[-1]), dtype=x.dtype, device=x.device)
    dev = _dev(x, out)
    cols = x.shape[-1]
    with torch.cuda.device(dev):
        check(lib.kllm_b200_select_last_row(_ptr(x), x.numel() // cols, cols, _ptr(out),
                                            dtype_code(x), _stream(dev)))
    return out


def select_last_rows(x: torch.Tensor, seq_len: int = 0, n_seqs: int | None = None,
                     seq_ends: torch.Tensor | None = None, out: torch.Tensor | None = None,
                     err_flags: torch.Tensor | None = None) -> torch.Tensor:
    cols = x.shape[-1]
    rows = x.numel() // cols
    if seq_ends is not None:
        n_seqs = seq_ends.numel()
    elif n_seqs is None:
        n_seqs = rows // seq_len
    if out is None:
        out = torch.empty((n_seqs, cols), dtype=x.dtype, device=x.device)
    dev = _dev(x, out, seq_ends, err_flags)
    with torch.cuda.device(dev):
        check(lib.kllm_b200_select_last_rows(_ptr(x), rows, cols, _ptr(seq_ends), seq_len, n_seqs,
                                             _ptr(out), dtype_code(x), _ptr(err_flags),
                                             _stream(dev)))
    return out


def attention_workspace_bytes(n_tokens: int, n_heads: int, n_kv_heads: int, head_dim: int,
                              max_seq: int) -> int:
    import ctypes
    n = ctypes.c_int64(0)
    check(lib.kllm_b200_attention_workspace_bytes(n_tokens, n_heads, n_kv_heads, head_dim, max_seq,
                                                  ctypes.addressof(n)))
    return n.value


def attention_head_major(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                         positions: torch.Tensor, slots: torch.Tensor, seq_len: int = 1,
                         out: torch.Tensor | None = None, workspace: torch.Tensor | None = None,
                         err_flags: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of q [T, Hq, D] over the head-major cache of one
    layer [n_slots, Hkv, max_seq, D]: token t sees positions 0..positions[t]
    of slot slots[t]. ``workspace=None`` allocates the preferred split
    workspace here, zero-filled (the C entry point itself never allocates; a
    caller-provided workspace must be zeroed once before its first use)."""
    T, Hq, D = q.shape
    n_slots, Hkv, max_seq, _ = k_cache.shape
    if out is None:
        out = torch.empty_like(q)
    if workspace is None:
        nbytes = attention_workspace_bytes(T, Hq, Hkv, D, max_seq)
        workspace = torch.zeros(max(nbytes, 16), dtype=torch.uint8, device=q.device)
    dev = _dev(q, k_cache, v_cache, positions, slots, out, workspace, err_flags)
    if positions.dtype != torch.int32 or slots.dtype != torch.int32:
        raise KllmError(_capi.ERR_DTYPE, "attention: positions and slots must be int32")
    with torch.cuda.device(dev):
        check(lib.kllm_b200_attention_head_major(
            _ptr(q), _ptr(k_cache), _ptr(v_cache), _ptr(out), _ptr(positions), _ptr(slots), T, seq_len, Hq,
            Hkv, D, n_slots, max_seq, dtype_code(q), _ptr(workspace), workspace.numel(), _ptr(err_flags),
            _stream(dev)))
    return out


def silu_mul(gate: torch.Tensor, up: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    if out is None:
        out = torch.empty_like(gate)
    dev = _dev(gate, up, out)
    if not (gate.numel() == up.numel() == out.numel()):
        raise KllmError(_capi.ERR_SHAPE, "silu_mul shape mismatch")
    if not (gate.dtype == up.dtype == out.dtype):
        raise KllmError(_capi.ERR_DTYPE, "silu_mul dtype mismatch")
    with torch.cuda.device(dev):
        check(lib.kllm_b200_silu_mul(_ptr(gate), _ptr(up), _ptr(out), gate.numel(),
                                     dtype_code(gate), _stream(dev)))
    return out


def _gemm_checks(x: torch.Tensor, weights, out: torch.Tensor, biases):
    if x.dim() != 2 or any(w.dim() != 2 for w in weights):
        raise KllmError(_capi.ERR_SHAPE, "linear: x and weights must be 2-D")
    if any(t.dtype != torch.float16 for t in (x, out, *weights)):
        raise KllmError(_capi.ERR_DTYPE, "linear: x, weights and out must be float16")
    n, k = weights[0].shape
    if x.shape[1] != k or any(w.shape != (n, k) for w in weights) or out.shape != (x.shape[0], n):
        raise KllmError(_capi.ERR_SHAPE, "linear shape mismatch")
    present = [b for b in biases if b is not None]
    if any(b.numel() != n for b in present):
        raise KllmError(_capi.ERR_SHAPE, "linear: bias length must equal the output columns")
    if len({b.dtype for b in present}) > 1:
        raise KllmError(_capi.ERR_DTYPE, "linear_swiglu: biases must share a dtype")
    return dtype_code(present[0]) if present else F16


def linear(x: torch.Tensor, w: torch.Tensor, bias: torch.Tensor | None = None,
           out: torch.Tensor | None = None, err_flags: torch.Tensor | None = None) -> torch.Tensor:
    """out = fp16(fp16(x @ w.T) + bias): the reference linear() (matmul +
    add_bias_inplace) as one tcgen05 GEMM. x [m, k], w [n, k] fp16."""
    if out is None:
        out = torch.empty(x.shape[0], w.shape[0], dtype=torch.float16, device=x.device)
    dev = _dev(x, w, bias, out, err_flags)
    bias_dtype = _gemm_checks(x, [w], out, [bias])
    with torch.cuda.device(dev):
        check(lib.kllm_b200_linear(_ptr(x), _ptr(w), _ptr(bias), bias_dtype, _ptr(out), x.shape[0],
                                   w.shape[0], x.shape[1], _ptr(err_flags), _stream(dev)))
    return out


def linear_swiglu(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor,
                  b_gate: torch.Tensor | None = None, b_up: torch.Tensor | None = None,
                  out: torch.Tensor | None = None, err_flags: torch.Tensor | None = None) -> torch.Tensor:
    """out = silu_mul(linear(x, w_gate, b_gate), linear(x, w_up, b_up)) in one
    kernel; w_gate and w_up [n, k] fp16."""
    if out is None:
        out = torch.empty(x.shape[0], w_gate.shape[0], dtype=torch.float16, device=x.device)
    dev = _dev(x, w_gate, w_up, b_gate, b_up, out, err_flags)
    bias_dtype = _gemm_checks(x, [w_gate, w_up], out, [b_gate, b_up])
    with torch.cuda.device(dev):
        check(lib.kllm_b200_linear_swiglu(_ptr(x), _ptr(w_gate), _ptr(w_up), _ptr(b_gate), _ptr(b_up),
                                          bias_dtype, _ptr(out), x.shape[0], w_gate.shape[0], x.shape[1],
                                          _ptr(err_flags), _stream(dev)))
    return out


def qkv_linear_rope_kv_append(x: torch.Tensor, wq: torch.Tensor, wk: torch.Tensor, wv: torch.Tensor,
                              bq: torch.Tensor | None, bk: torch.Tensor | None, bv: torch.Tensor | None,
                              positions: torch.Tensor, slots: torch.Tensor, theta: float,
                              k_cache: torch.Tensor, v_cache: torch.Tensor, q_out: torch.Tensor | None = None,
                              err_flags: torch.Tensor | None = None) -> torch.Tensor:
    """q = rope(x @ wq.T + bq) into q_out [T, Hq*D]; k = rope(x @ wk.T + bk) and
    v = x @ wv.T + bv appended to the caches [n_slots, Hkv, max_seq, D] (one
    tcgen05 GEMM with the bias + RoPE + KV append in its epilogue)."""
    n_slots, Hkv, max_seq, D = k_cache.shape
    Hq = wq.shape[0] // D
    if q_out is None:
        q_out = torch.empty(x.shape[0], wq.shape[0], dtype=torch.float16, device=x.device)
    dev = _dev(x, wq, wk, wv, bq, bk, bv, positions, slots, k_cache, v_cache, q_out, err_flags)
    bias = next((b for b in (bq, bk, bv) if b is not None), None)
    bias_dtype = dtype_code(bias) if bias is not None else F16
    with torch.cuda.device(dev):
        check(lib.kllm_b200_qkv_linear_rope_kv_append(
            _ptr(x), _ptr(wq), _ptr(wk), _ptr(wv), _ptr(bq), _ptr(bk), _ptr(bv), bias_dtype, _ptr(positions),
            _ptr(slots), x.shape[0], x.shape[1], Hq, Hkv, D, theta, _ptr(q_out), _ptr(k_cache), _ptr(v_cache),
            n_slots, max_seq, _ptr(err_flags), _stream(dev)))
    return q_out


def rope_inplace(x: torch.Tensor, past_len: int, theta: float) -> torch.Tensor:
    """x [seq, heads, head_dim] rotated in place at positions past_len + t."""
    dev = _dev(x)
    seq, heads, head_dim = x.shape
    with torch.cuda.device(dev):
        check(lib.kllm_b200_rope_inplace(_ptr(x), seq, heads, head_dim, past_len, theta,
                                         dtype_code(x), _stream(dev)))
    return x


def copy_kv_to_cache(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor,
                     v_cache: torch.Tensor, past_len: int) -> None:
    """k/v [seq, kv_heads, head_dim] -> caches [max_seq, kv_heads, head_dim] at past_len."""
    dev = _dev(k, v, k_cache, v_cache)
    seq, kv_heads, head_dim = k.shape
    with torch.cuda.device(dev):
        check(lib.kllm_b200_copy_kv_to_cache(_ptr(k), _ptr(v), seq, kv_heads, head_dim,
                                             _ptr(k_cache), _ptr(v_cache), k_cache.shape[0],
                                             past_len, dtype_code(k), dtype_code(k_cache),
                                             _stream(dev)))


def qkv_bias_rope_kv_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                            bq: torch.Tensor | None, bk: torch.Tensor | None,
                            bv: torch.Tensor | None, positions: torch.Tensor,
                            slots: torch.Tensor, theta: float, k_cache: torch.Tensor,
                            v_cache: torch.Tensor,
                            err_flags: torch.Tensor | None = None) -> None:
    """q [T, Hq, D] rotated in place; k/v [T, Hkv, D] appended (rotated /
    biased) into caches [n_slots, Hkv, max_seq, D]."""
    dev = _dev(q, k, v, bq, bk, bv, positions, slots, k_cache, v_cache, err_flags)
    T, Hq, D = q.shape
    Hkv = k.shape[1]
    bias = next((b for b in (bq, bk, bv) if b is not None), None)
    bias_dtype = dtype_code(bias) if bias is not None else F16
    with torch.cuda.device(dev):
        check(lib.kllm_b200_qkv_bias_rope_kv_append(
            _ptr(q), _ptr(k), _ptr(v), _ptr(bq), _ptr(bk), _ptr(bv), bias_dtype, _ptr(positions),
            _ptr(slots), T, Hq, Hkv, D, theta, _ptr(k_cache), _ptr(v_cache), k_cache.shape[0],
            k_cache.shape[2], _ptr(err_flags), _stream(dev)))


def dequantize_int8(data: torch.Tensor, scale: torch.Tensor,
                    out_dtype: torch.dtype = torch.float16,
                    out: torch.Tensor | None = None) -> torch.Tensor:
    """out = data * scale[0]; fp16 output rounds like the reference weight loader."""
    if out is None:
        out = torch.empty(data.shape, dtype=out_dtype, device=data.device)
    dev = _dev(data, scale, out)
    if data.dtype != torch.int8 or scale.dtype != torch.float32:
        raise KllmError(_capi.ERR_DTYPE, "dequantize_int8 expects int8 data and an fp32 scale")
    with torch.cuda.device(dev):
        check(lib.kllm_b200_dequantize_int8(_ptr(data), _ptr(scale), _ptr(out), data.numel(),
                                            dtype_code(out), _stream(dev)))
    return out


def dequantize_int8_rne(data: torch.Tensor, scale: torch.Tensor, out: torch.Tensor | None = None,
                        mismatches: torch.Tensor | None = None) -> torch.Tensor:
    """out = data * scale[0] in fp16 rounded to nearest even (IEEE), not by
    the reference loader's rounding; when given, ``mismatches`` (a CUDA int64
    tensor of one element) is increased by the number of elements where the
    two roundings differ."""
    if out is None:
        out = torch.empty(data.shape, dtype=torch.float16, device=data.device)
    dev = _dev(data, scale, out, mismatches)
    if data.dtype != torch.int8 or scale.dtype != torch.float32 or out.dtype != torch.float16:
        raise KllmError(_capi.ERR_DTYPE, "dequantize_int8_rne expects int8 data, an fp32 scale and fp16 out")
    if mismatches is not None and (mismatches.dtype != torch.int64 or mismatches.numel() != 1):
        raise KllmError(_capi.ERR_DTYPE, "dequantize_int8_rne: mismatches must be one int64")
    with torch.cuda.device(dev):
        check(lib.kllm_b200_dequantize_int8_rne(_ptr(data), _ptr(scale), _ptr(out), data.numel(), _ptr(mismatches),
                                                _stream(dev)))
    return out


def dequantize_int8_batched(data: list[torch.Tensor], scales: list[torch.Tensor],
                            outs: list[torch.Tensor]) -> list[torch.Tensor]:
    """outs[i] = data[i] * scales[i][0] for every i in one launch (rounding
    as in dequantize_int8 for the outputs' dtype, which must all match)."""
    import ctypes
    n = len(data)
    if not (len(scales) == len(outs) == n):
        raise KllmError(_capi.ERR_SHAPE, "dequantize_int8_batched: list lengths differ")
    if n == 0:
        return outs
    dev = _dev(*data, *scales, *outs)
    out_dtypes = {dtype_code(o) for o in outs}
    if len(out_dtypes) != 1:
        raise KllmError(_capi.ERR_DTYPE, "dequantize_int8_batched: outputs must share one dtype")
    for d, sc, o in zip(data, scales, outs):
        if d.dtype != torch.int8 or sc.dtype != torch.float32 or d.numel() != o.numel():
            raise KllmError(_capi.ERR_DTYPE, "dequantize_int8_batched: int8 data, fp32 scale, matching sizes")
    arr = ctypes.c_void_p * n
    d_arr = arr(*[d.data_ptr() for d in data])
    s_arr = arr(*[sc.data_ptr() for sc in scales])
    o_arr = arr(*[o.data_ptr() for o in outs])
    c_arr = (ctypes.c_int64 * n)(*[d.numel() for d in data])
    with torch.cuda.device(dev):
        check(lib.kllm_b200_dequantize_int8_batched(d_arr, s_arr, o_arr, c_arr, n, out_dtypes.pop(),
                                                    _stream(dev)))
    return outs


# ---- paged KV cache ---------------------------------------------------------


def _call(device, entry, *args) -> None:
    """Calls a C entry point with `device` current (the context is entered only
    when it is not) and its stream appended, and checks the status."""
    index = device.index
    if index == _current_device():
        status = entry(*args, _raw_stream(index))
    else:
        with torch.cuda.device(device):
            status = entry(*args, _stream(device))
    if status != _capi.OK:
        check(status)


def _all_on(device, *tensors) -> None:
    """Checks that every given tensor is contiguous and on `device`."""
    index = device.index
    for t in tensors:
        if t is not None and (t.get_device() != index or not t.is_contiguous()):
            _dev(t)  # not a CUDA tensor, not contiguous
            raise KllmError(_capi.ERR_INVALID_ARG, "tensors are on different devices")


def _flags(device, err_flags) -> None:
    """Checks an optional flag word: int32 on `device`."""
    if err_flags is not None:
        if err_flags.dtype is not torch.int32:
            raise KllmError(_capi.ERR_DTYPE, "err_flags must be int32")
        _all_on(device, err_flags)


class PagedKVCache:
    """One layer's paged KV cache (kllm_b200_paged_cache) over given tensors.

    k_pages and v_pages [n_pages, n_kv_heads, page_size, head_dim], fp16 or
    int8 (codes; then k_scales and v_scales, fp32 [n_pages, n_kv_heads,
    page_size], hold the value of one code step per row); page_table int32
    [n_seqs, max_pages] names the page of each page_size positions of each
    sequence. head_dim 64 or 128, page_size a power of two of at least 8. The
    tensors stay the caller's: write page_table in place to hand out pages."""

    def __init__(self, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                 k_scales: torch.Tensor | None = None, v_scales: torch.Tensor | None = None):
        self.device = _dev(k_pages, v_pages, page_table, k_scales, v_scales)
        if k_pages.dim() != 4 or v_pages.shape != k_pages.shape or page_table.dim() != 2:
            raise KllmError(_capi.ERR_SHAPE, "paged cache: k_pages and v_pages [n_pages, n_kv_heads, page_size, "
                                             "head_dim], page_table [n_seqs, max_pages]")
        if k_pages.dtype not in (torch.float16, torch.int8) or v_pages.dtype != k_pages.dtype:
            raise KllmError(_capi.ERR_DTYPE, "paged cache: pages must both be float16 or both int8")
        if page_table.dtype != torch.int32:
            raise KllmError(_capi.ERR_DTYPE, "paged cache: page_table must be int32")
        scales = (k_scales, v_scales)
        if k_pages.dtype == torch.int8:
            if any(s is None or s.dtype != torch.float32 for s in scales):
                raise KllmError(_capi.ERR_DTYPE, "paged cache: int8 pages need float32 k_scales and v_scales")
            if any(s.shape != k_pages.shape[:3] for s in scales):
                raise KllmError(_capi.ERR_SHAPE, "paged cache: scales must be [n_pages, n_kv_heads, page_size]")
        elif any(s is not None for s in scales):
            raise KllmError(_capi.ERR_INVALID_ARG, "paged cache: float16 pages take no scales")
        self._tensors = (k_pages, v_pages, k_scales, v_scales, page_table)
        self._workspace_bytes: dict[tuple[int, int], int] = {}  # of attention_paged, by (tokens, query heads)
        n_pages, n_kv_heads, page_size, head_dim = k_pages.shape
        n_seqs, max_pages = page_table.shape
        self._descriptor = _capi.PagedCache(None, None, None, None, None, n_pages, page_size, n_kv_heads, head_dim,
                                            n_seqs, max_pages, dtype_code(k_pages))

    k_pages = property(lambda self: self._tensors[0])
    v_pages = property(lambda self: self._tensors[1])
    k_scales = property(lambda self: self._tensors[2])
    v_scales = property(lambda self: self._tensors[3])
    page_table = property(lambda self: self._tensors[4])

    @classmethod
    def allocate(cls, n_pages: int, page_size: int, n_kv_heads: int, head_dim: int, n_seqs: int, max_pages: int,
                 dtype: torch.dtype = torch.float16, device="cuda") -> "PagedKVCache":
        """An empty cache: zero pages, every table entry -1 (no page)."""
        shape = (n_pages, n_kv_heads, page_size, head_dim)
        pages = [torch.zeros(shape, dtype=dtype, device=device) for _ in range(2)]
        scales = [torch.zeros(shape[:3], dtype=torch.float32, device=device) if dtype == torch.int8 else None
                  for _ in range(2)]
        table = torch.full((n_seqs, max_pages), -1, dtype=torch.int32, device=device)
        return cls(*pages, table, *scales)

    def descriptor(self) -> _capi.PagedCache:
        """The C descriptor (kllm_b200_paged_cache) of the tensors."""
        d = self._descriptor
        k, v, ks, vs, table = self._tensors
        d.k_pages, d.v_pages, d.page_table = k.data_ptr(), v.data_ptr(), table.data_ptr()
        if ks is not None:
            d.k_scales, d.v_scales = ks.data_ptr(), vs.data_ptr()
        return d


def _head_rows(x: torch.Tensor, heads: int | None, head_dim: int, device, what: str) -> int:
    """Checks x [n_tokens, heads, head_dim] on `device`, fp16 with contiguous
    heads, and returns the elements between its tokens (views into one packed
    projection pass)."""
    shape, stride = x.shape, x.stride()
    if (x.dtype is not torch.float16 or x.get_device() != device.index or len(shape) != 3 or shape[2] != head_dim
            or (heads is not None and shape[1] != heads) or stride[2] != 1
            or (stride[1] != head_dim and shape[1] > 1)):
        if x.get_device() != device.index:
            raise KllmError(_capi.ERR_INVALID_ARG,
                            "tensors are on different devices" if x.is_cuda else "expected a CUDA tensor")
        if x.dtype != torch.float16:
            raise KllmError(_capi.ERR_DTYPE, f"{what}: q, k, v and outputs must be float16")
        if len(shape) != 3 or shape[2] != head_dim or (heads is not None and shape[1] != heads):
            raise KllmError(_capi.ERR_SHAPE, f"{what}: expected [n_tokens, heads, {head_dim}], got {tuple(shape)}")
        raise KllmError(_capi.ERR_SHAPE, f"{what}: the heads of a token must be contiguous")
    return stride[0] if shape[0] > 1 else shape[1] * head_dim  # the stride of a single token is never used


def _token_index(n: int, device, what: str, *tensors) -> None:
    """Checks positions, seqs, slots or tokens: int32 [n] on `device`, contiguous."""
    for x in tensors:
        if x is not None and (x.dtype is not torch.int32 or x.dim() != 1 or x.shape[0] != n
                              or x.get_device() != device.index or not x.is_contiguous()):
            if x.dtype != torch.int32:
                raise KllmError(_capi.ERR_DTYPE, f"{what}: positions, seqs, slots and tokens must be int32")
            if x.shape != (n,):
                raise KllmError(_capi.ERR_SHAPE, f"{what}: positions, seqs, slots and tokens must hold one entry each")
            _all_on(device, x)


def _parameters(expected, names: str, what: str) -> int:
    """Checks optional (tensor, number of values) pairs and returns their dtype's code."""
    dtype = None
    for x, n in expected:
        if x is None:
            continue
        if x.numel() != n:
            raise KllmError(_capi.ERR_SHAPE, f"{what}: {names} must hold {n} values, got {x.numel()}")
        if dtype is not None and x.dtype != dtype:
            raise KllmError(_capi.ERR_DTYPE, f"{what}: {names} must share a dtype")
        dtype = x.dtype
    return F16 if dtype is None else _DTYPES.get(dtype, -1)  # -1: refused by the library


def qkv_norm_rope_kv_append_paged(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cache: PagedKVCache,
                                  positions: torch.Tensor, seqs: torch.Tensor, theta: float,
                                  bq: torch.Tensor | None = None, bk: torch.Tensor | None = None,
                                  bv: torch.Tensor | None = None, q_norm: torch.Tensor | None = None,
                                  k_norm: torch.Tensor | None = None, eps: float = 1e-6,
                                  q_out: torch.Tensor | None = None,
                                  err_flags: torch.Tensor | None = None) -> torch.Tensor:
    """Bias, per-head RMSNorm of q and k (with the weights q_norm and k_norm
    [head_dim]; None: no norm) and rotate-half RoPE; k and v are appended to
    the paged cache at row positions[t] of sequence seqs[t], q goes to q_out
    (None: rotated in place). q [T, Hq, D], k and v [T, Hkv, D] fp16, tokens
    at any stride that is a multiple of 8. positions[t] == -1 is padding. No
    two tokens of one call may write the same row of a page."""
    what = "qkv_norm_rope_kv_append_paged"
    c, dev = cache.descriptor(), cache.device
    D, Hkv = c.head_dim, c.n_kv_heads
    if q_out is None:
        q_out = q
    sq = _head_rows(q, None, D, dev, what)
    T, Hq, _ = q.shape
    so = sq if q_out is q else _head_rows(q_out, Hq, D, dev, what)
    sk, sv = _head_rows(k, Hkv, D, dev, what), _head_rows(v, Hkv, D, dev, what)
    if not (k.shape[0] == v.shape[0] == q_out.shape[0] == T):
        raise KllmError(_capi.ERR_SHAPE, f"{what}: q, k, v and q_out must hold the same number of tokens")
    _token_index(T, dev, what, positions, seqs)
    _all_on(dev, bq, bk, bv, q_norm, k_norm)
    _flags(dev, err_flags)
    bias = norm = F16
    if bq is not None or bk is not None or bv is not None:
        bias = _parameters(((bq, Hq * D), (bk, Hkv * D), (bv, Hkv * D)), "biases", what)
    if q_norm is not None or k_norm is not None:
        norm = _parameters(((q_norm, D), (k_norm, D)), "norm weights", what)
    _call(dev, lib.kllm_b200_qkv_norm_rope_kv_append_paged, q.data_ptr(), sq, k.data_ptr(), sk, v.data_ptr(), sv,
          _ptr(bq), _ptr(bk), _ptr(bv), bias, _ptr(q_norm), _ptr(k_norm), norm, eps, theta, positions.data_ptr(),
          seqs.data_ptr(), T, Hq, c, q_out.data_ptr(), so, _ptr(err_flags))
    return q_out


def kv_read_paged(cache: PagedKVCache, positions: torch.Tensor, seqs: torch.Tensor,
                  k_out: torch.Tensor | None = None, v_out: torch.Tensor | None = None,
                  out_slots: torch.Tensor | None = None,
                  err_flags: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """The cached rows at positions[t] of sequences seqs[t] as fp16. Without
    out_slots: token rows [T, Hkv, D] (allocated as zeros when not given).
    With out_slots: row positions[t] of slot out_slots[t] of the head-major
    caches k_out and v_out [n_slots, Hkv, max_seq, D], which
    attention_head_major reads. Rows of padding (position -1) are not written."""
    what = "kv_read_paged"
    c, dev = cache.descriptor(), cache.device
    T = positions.numel()
    _token_index(T, dev, what, positions, seqs, out_slots)
    if out_slots is None:
        shape, n_slots, max_seq = (T, c.n_kv_heads, c.head_dim), 0, 0
        if k_out is None:
            k_out = torch.zeros(shape, dtype=torch.float16, device=dev)
        if v_out is None:
            v_out = torch.zeros(shape, dtype=torch.float16, device=dev)
    else:
        if k_out is None or v_out is None or k_out.dim() != 4:
            raise KllmError(_capi.ERR_SHAPE, f"{what}: out_slots needs k_out and v_out [n_slots, kv_heads, max_seq, "
                                             "head_dim]")
        n_slots, _, max_seq, _ = k_out.shape
        shape = (n_slots, c.n_kv_heads, max_seq, c.head_dim)
    if k_out.shape != shape or v_out.shape != shape:
        raise KllmError(_capi.ERR_SHAPE, f"{what}: outputs must be {shape}")
    if k_out.dtype != torch.float16 or v_out.dtype != torch.float16:
        raise KllmError(_capi.ERR_DTYPE, f"{what}: outputs must be float16")
    _all_on(dev, k_out, v_out)
    _flags(dev, err_flags)
    _call(dev, lib.kllm_b200_kv_read_paged, c, positions.data_ptr(), seqs.data_ptr(), T, _ptr(out_slots), n_slots,
          max_seq, k_out.data_ptr(), v_out.data_ptr(), _ptr(err_flags))
    return k_out, v_out


def attention_paged_workspace_bytes(n_tokens: int, n_heads: int, cache: PagedKVCache) -> int:
    n = ctypes.c_int64(0)
    if cache.device.index == _current_device():
        check(lib.kllm_b200_attention_paged_workspace_bytes(n_tokens, n_heads, cache.descriptor(), n))
    else:
        with torch.cuda.device(cache.device):
            check(lib.kllm_b200_attention_paged_workspace_bytes(n_tokens, n_heads, cache.descriptor(), n))
    return n.value


def attention_paged(q: torch.Tensor, cache: PagedKVCache, positions: torch.Tensor, seqs: torch.Tensor,
                    out: torch.Tensor | None = None, workspace: torch.Tensor | None = None,
                    err_flags: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of single new tokens over the paged cache: token t sees
    positions 0..positions[t] of sequence seqs[t]; q and out [T, Hq, D] fp16,
    tokens at any stride that is a multiple of 8. Padding rows (position -1)
    become zeros. out must not overlap q. ``workspace=None`` allocates the
    preferred one here (the C entry point itself never allocates); a given one
    needs no clearing and serves one call at a time, captured ones included."""
    what = "attention_paged"
    c, dev = cache.descriptor(), cache.device
    sq = _head_rows(q, None, c.head_dim, dev, what)
    T, Hq, D = q.shape
    if out is None:
        out = torch.empty((T, Hq, D), dtype=q.dtype, device=dev)
    so = _head_rows(out, Hq, D, dev, what)
    if out.shape[0] != T:
        raise KllmError(_capi.ERR_SHAPE, f"{what}: q and out must hold the same number of tokens")
    _token_index(T, dev, what, positions, seqs)
    _all_on(dev, workspace)
    _flags(dev, err_flags)
    nbytes = 0
    if workspace is not None:
        nbytes = workspace.numel() * workspace.element_size()
    elif c.max_pages * c.page_size >= _capi.PAGED_SPLIT_MIN:
        nbytes = cache._workspace_bytes.get((T, Hq))
        if nbytes is None:
            nbytes = cache._workspace_bytes[T, Hq] = attention_paged_workspace_bytes(T, Hq, cache)
        if nbytes:
            workspace = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    _call(dev, lib.kllm_b200_attention_paged, q.data_ptr(), sq, c, positions.data_ptr(), seqs.data_ptr(), T, Hq,
          out.data_ptr(), so, workspace.data_ptr() if nbytes else None, nbytes, _ptr(err_flags))
    return out


# ---- log probabilities --------------------------------------------------------


class TokenLogprobs(NamedTuple):
    """What token_logprobs answers for each row of logits."""
    logprobs: torch.Tensor | None       # fp32 [rows]: log probability of the given token
    ranks: torch.Tensor | None          # int32 [rows]: 1 + the logits above it
    entropies: torch.Tensor             # fp32 [rows]
    top_ids: torch.Tensor | None        # int32 [rows, top_k], most likely first
    top_logprobs: torch.Tensor | None   # fp32 [rows, top_k]


def token_logprobs_buffers(logits: torch.Tensor, top_k: int = 0, tokens: bool = True) -> TokenLogprobs:
    """Outputs for token_logprobs on logits of this shape."""
    rows, dev = logits.shape[0], logits.device

    def make(dtype, *shape):
        return torch.empty(shape, dtype=dtype, device=dev)

    return TokenLogprobs(make(torch.float32, rows) if tokens else None, make(torch.int32, rows) if tokens else None,
                         make(torch.float32, rows), make(torch.int32, rows, top_k),
                         make(torch.float32, rows, top_k))


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor | None = None, top_k: int = 0,
                   out: TokenLogprobs | None = None, err_flags: torch.Tensor | None = None) -> TokenLogprobs:
    """Log probability and rank of tokens[r] (int32; -1: none asked) under each
    row of logits [rows, vocab] (fp16 or fp32, rows at any stride), the row's
    entropy, and its top_k (0 to 32) largest logits as ids and log
    probabilities, equal logits in the order of their ids. Outputs given in
    ``out`` that nothing asks for (logprobs and ranks without tokens) stay as
    they were."""
    what = "token_logprobs"
    dev = logits.device
    if not logits.is_cuda:
        raise KllmError(_capi.ERR_INVALID_ARG, "expected a CUDA tensor")
    if logits.dim() != 2 or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise KllmError(_capi.ERR_SHAPE, f"{what}: logits must be [rows, vocab] with contiguous rows")
    rows, vocab = logits.shape
    dtype = dtype_code(logits)
    if not 0 <= top_k <= min(32, vocab):
        raise KllmError(_capi.ERR_SHAPE, f"{what}: top_k {top_k} must be 0 to 32 and at most vocab")
    if out is None:
        out = token_logprobs_buffers(logits, top_k, tokens is not None)
    logprobs, ranks, entropies, top_ids, top_logprobs = out
    if tokens is not None:
        _token_index(rows, dev, what, tokens)
        if logprobs is None or ranks is None:
            raise KllmError(_capi.ERR_INVALID_ARG, f"{what}: tokens need logprobs and ranks among the outputs")
    _all_on(dev, logprobs, ranks, entropies, top_ids, top_logprobs)
    _flags(dev, err_flags)
    for t, kind, shape in ((logprobs, torch.float32, (rows,)), (ranks, torch.int32, (rows,)),
                           (entropies, torch.float32, (rows,)), (top_ids, torch.int32, (rows, top_k)),
                           (top_logprobs, torch.float32, (rows, top_k))):
        if t is not None and (t.dtype != kind or t.shape != shape):
            raise KllmError(_capi.ERR_SHAPE, f"{what}: an output has another shape or dtype than {shape}, {kind}")
    asked = tokens is not None
    _call(dev, lib.kllm_b200_token_logprobs, logits.data_ptr(), dtype, rows, vocab,
          logits.stride(0) if rows > 1 else vocab, _ptr(tokens), _ptr(logprobs) if asked else None,
          _ptr(ranks) if asked else None, _ptr(entropies), top_k, _ptr(top_ids) if top_k else None,
          _ptr(top_logprobs) if top_k else None, _ptr(err_flags))
    return out
