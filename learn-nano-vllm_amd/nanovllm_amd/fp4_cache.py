"""The 4-bit key/value cache: 4.5 bits per value where the 16-bit caches take 16.

``Fp4Cache`` stands in the place of a layer's ``k_cache`` or ``v_cache`` tensor wherever the package
takes one: ``store_kvcache`` quantises the rows that it scatters (the reference's store,
nanovllm/layers/attention.py:33-40), ``paged_decode``, ``varlen_prefill``,
``flash_attn_with_kvcache`` and ``flash_attn_varlen_func`` read the codes, and ``Attention`` and
``attention_with_prologue`` do both.  ``load_kvcache`` gives the rows back.  The reference has
no such cache.
"""
from __future__ import annotations

import functools
from typing import NamedTuple

import torch

from nanovllm_amd import _lib

GROUP = 32    # dimensions that share a scale


class Fp4Cache(NamedTuple):
    """One layer's keys or values in 4 bits.

    data   uint8   [num_blocks, num_kv_heads, block_size, head_dim / 2], two e2m1 codes a byte
    scale  float16 [num_blocks, num_kv_heads, head_dim / 32, block_size], one for 32 dimensions

    A value stands for code * scale, scale = max |x| / 6 of its 32 dimensions in float16, code the
    nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives (ties to the even code).  Groups
    with an infinity or NaN read back as NaN.  include/nvk.h has the order of a row's codes, which
    differs between keys and values: a cache of keys cannot be read as one of values.
    head_dim is 128 or 64, block_size a multiple of 16.
    """
    data: torch.Tensor
    scale: torch.Tensor

    @classmethod
    def zeros(cls, num_blocks: int, block_size: int, num_kv_heads: int, head_dim: int,
              device="cuda") -> "Fp4Cache":
        """A cache of zeros."""
        if head_dim not in (64, 128) or block_size <= 0 or block_size % 16:
            raise _lib.NvkError("a 4-bit cache has head_dim 128 or 64 and pages of a multiple of 16 "
                                f"tokens, got {head_dim} and {block_size}")
        return cls(torch.zeros(num_blocks, num_kv_heads, block_size, head_dim // 2,
                               dtype=torch.uint8, device=device),
                   torch.zeros(num_blocks, num_kv_heads, head_dim // GROUP, block_size,
                               dtype=torch.float16, device=device))

    def numel(self) -> int:
        """Values that the cache holds (Attention takes a cache of none for none at all)."""
        return 2 * self.data.numel()


def _check_caches(k_cache, v_cache):
    """(num_blocks, block_size, num_kv_heads, head_dim) of a pair of caches."""
    if not (isinstance(k_cache, Fp4Cache) and isinstance(v_cache, Fp4Cache)):
        raise _lib.NvkError("k_cache and v_cache must both be Fp4Cache")
    (kd, ks), (vd, vs) = k_cache, v_cache
    shape = kd.shape
    if ((kd.dtype, vd.dtype, ks.dtype, vs.dtype) != _CACHE_DTYPES or len(shape) != 4
            or not (kd.is_contiguous() and vd.is_contiguous() and ks.is_contiguous()
                    and vs.is_contiguous())):
        raise _lib.NvkError("Fp4Cache must be contiguous uint8 [num_blocks, Hkv, block_size, D / 2] "
                            "and float16 [num_blocks, Hkv, D / 32, block_size]")
    nb, hkv, bs, half = shape
    if ((half != 64 and half != 32) or bs % 16 or vd.shape != shape
            or not ks.shape == vs.shape == (nb, hkv, half // 16, bs)):
        raise _lib.NvkError("Fp4Cache shapes disagree, or head_dim is not 128 or 64, or block_size "
                            "not a multiple of 16")
    return nb, bs, hkv, 2 * half


_CACHE_DTYPES = (torch.uint8, torch.uint8, torch.float16, torch.float16)


def _device(k_cache, v_cache, *tensors):
    """The GPU that the caches and the tensors are on (they have to share one)."""
    (kd, ks), (vd, vs) = k_cache, v_cache
    gpu = kd.get_device()
    if not 0 <= gpu == ks.get_device() == vd.get_device() == vs.get_device():
        _lib.require_gpu(kd, ks, vd, vs)    # raises
    for t in tensors:
        if t.get_device() != gpu:
            _lib.require_gpu(kd, t)         # raises
    return kd.device


_ROWS = {torch.bfloat16: _lib.NVK_DTYPE_BF16, torch.float16: _lib.NVK_DTYPE_F16}


def _rows_dtype(dtype: torch.dtype) -> int:
    code = _ROWS.get(dtype)
    if code is None:
        raise _lib.NvkError(f"a 4-bit cache takes and gives bfloat16 and float16 rows, got {dtype}")
    return code


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(*sizes: int) -> int:
    """nvk_fp4_attention_workspace_size, a function of its sizes alone."""
    return _lib.load().nvk_fp4_attention_workspace_size(*sizes)


def fp4_store(key: torch.Tensor, value: torch.Tensor, k_cache: Fp4Cache, v_cache: Fp4Cache,
              slot_mapping: torch.Tensor) -> None:
    """``store_kvcache`` into 4-bit caches: the same arguments and checks; rows bf16 or f16, 16-byte
    aligned."""
    nb, bs, hkv, d = _check_caches(k_cache, v_cache)
    dtype = _rows_dtype(key.dtype)
    N = key.shape[0]
    assert key.shape == value.shape == (N, hkv, d) and key.dtype == value.dtype
    ks, *k_inner = key.stride()
    vs, *v_inner = value.stride()
    assert k_inner == v_inner == [d, 1]
    assert slot_mapping.numel() == N
    dev = _device(k_cache, v_cache, key, value, slot_mapping)
    slots = _lib.int32(slot_mapping)
    with _lib.on_device(dev):
        code = _lib.load().nvk_fp4_store(
            key.data_ptr(), ks, value.data_ptr(), vs, k_cache.data.data_ptr(),
            k_cache.scale.data_ptr(), v_cache.data.data_ptr(), v_cache.scale.data_ptr(),
            slots.data_ptr(), N, hkv, d, bs, nb, dtype, _lib.stream_ptr(dev))
    if code:
        _lib.check(code)


def load_kvcache(k_cache: Fp4Cache, v_cache: Fp4Cache, slot_mapping: torch.Tensor,
                 dtype: torch.dtype = torch.bfloat16) -> tuple[torch.Tensor, torch.Tensor]:
    """The keys and values that 4-bit caches hold at the slots, [N, num_kv_heads, head_dim] of
    ``dtype`` (bfloat16 or float16) each: what ``store_kvcache`` with the same slots stored, as it
    was rounded.  A slot outside the cache (-1) gives zeros."""
    nb, bs, hkv, d = _check_caches(k_cache, v_cache)
    code = _rows_dtype(dtype)
    dev = _device(k_cache, v_cache, slot_mapping)
    slots = _lib.int32(slot_mapping)
    N = slots.numel()
    key = torch.empty((N, hkv, d), dtype=dtype, device=dev)
    value = torch.empty_like(key)
    with _lib.on_device(dev):
        st = _lib.load().nvk_fp4_load(
            k_cache.data.data_ptr(), k_cache.scale.data_ptr(), v_cache.data.data_ptr(),
            v_cache.scale.data_ptr(), slots.data_ptr(), N, hkv, d, bs, nb, key.data_ptr(), hkv * d,
            value.data_ptr(), hkv * d, code, _lib.stream_ptr(dev))
    if st:
        _lib.check(st)
    return key, value


def fp4_attention(q: torch.Tensor, k_cache: Fp4Cache, v_cache: Fp4Cache, seqlens_k: torch.Tensor,
                  block_table: torch.Tensor, softmax_scale=None, cu_seqlens_q=None,
                  max_seqlen_q: int = 1, max_seqlen_k: int | None = None,
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of q [tokens, Hq, D] over 4-bit caches.  Without ``cu_seqlens_q`` every
    sequence has ``max_seqlen_q`` queries and ``seqlens_k`` [B] keys (q may then be
    [B, max_seqlen_q, Hq, D]); with it both are prefix sums [B + 1].  The queries are the last of
    their sequence's keys.  ``max_seqlen_k`` bounds the keys of a sequence (None: what the block
    table holds).  Returns a tensor like q (or fills ``out``)."""
    nb, bs, hkv, d = _check_caches(k_cache, v_cache)
    dtype = _rows_dtype(q.dtype)
    shape, strides = q.shape, q.stride()
    if len(shape) == 3:
        tq, hq, dq = shape
        row, head, last = strides
    elif len(shape) == 4 and cu_seqlens_q is None and out is None and shape[1] == max_seqlen_q:
        b, n, hq, dq = shape
        tq = b * n
        seq, row, head, last = strides
        if n == 1:
            row = seq
        elif seq != n * row:
            q = q.contiguous()
            row, head, last = q.stride()[1:]
    else:
        raise _lib.NvkError("q must be [tokens, heads, head_dim]")
    if last != 1 or dq != d:
        raise _lib.NvkError("q must have unit last stride and the caches' head_dim")
    lens, bt = _lib.int32(seqlens_k), _lib.int32(block_table)
    cu_q = None if cu_seqlens_q is None else _lib.int32(cu_seqlens_q)
    batch = lens.numel()
    if cu_q is not None:
        if cu_q.numel() != batch:
            raise _lib.NvkError("cu_seqlens_q and cu_seqlens_k disagree on the batch size")
        batch -= 1
    elif batch * max_seqlen_q != tq:
        raise _lib.NvkError("q and cache_seqlens disagree on the batch size")
    if bt.dim() != 2 or len(bt) != batch:
        raise _lib.NvkError("block_table must be [batch, max_blocks]")
    dev = _device(k_cache, v_cache, q, lens, bt, lens if cu_q is None else cu_q)
    if out is None:
        out_row, out_head = hq * d, d
        out = torch.empty_like(q) if (row == out_row or tq < 2) and head == d else \
            torch.empty(shape, dtype=q.dtype, device=dev)
    else:
        if out.shape != shape or out.dtype != q.dtype or out.device != dev or out.stride(-1) != 1:
            raise _lib.NvkError("out must be like q, with unit last stride")
        out_row, out_head = out.stride()[:2]
    scale = d ** -0.5 if softmax_scale is None else float(softmax_scale)
    mq, mk, width = int(max_seqlen_q), int(max_seqlen_k or 0), bt.size(1)
    ws_bytes = _workspace_bytes(batch, mq, mk, hq, hkv, d, bs, width)
    with _lib.on_device(dev):
        stream = _lib.stream_ptr(dev)
        ws = _lib.workspace_on(dev, stream, ws_bytes)
        code = _lib.load().nvk_fp4_attention(
            q.data_ptr(), row, head, tq, k_cache.data.data_ptr(), k_cache.scale.data_ptr(),
            v_cache.data.data_ptr(), v_cache.scale.data_ptr(), _lib.ptr(cu_q), lens.data_ptr(),
            batch, mq, mk, bt.data_ptr(), width, width, bs, nb, hq, hkv, d, scale,
            out.data_ptr(), out_row, out_head, _lib.ptr(ws), ws_bytes, dtype, stream)
    if code:
        _lib.check(code)
    return out
