"""The 4-bit key/value cache: 4.5 bits per value where the 16-bit caches take 16.

``Fp4Cache`` stands in the place of a layer's ``k_cache`` or ``v_cache`` tensor wherever the package
takes one: ``store_kvcache`` quantises the rows that it scatters (the reference's store,
nanovllm/layers/attention.py:33-40), ``paged_decode``, ``varlen_prefill``,
``flash_attn_with_kvcache`` and ``flash_attn_varlen_func`` read the codes, and ``Attention`` and
``attention_with_prologue`` do both.  ``load_kvcache`` gives the rows back.  The reference has
no such cache.
"""
from __future__ import annotations

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
    for c in (k_cache, v_cache):
        if not isinstance(c, Fp4Cache):
            raise _lib.NvkError("k_cache and v_cache must both be Fp4Cache")
        if (c.data.dim() != 4 or c.scale.dim() != 4 or c.data.dtype != torch.uint8
                or c.scale.dtype != torch.float16 or not c.data.is_contiguous()
                or not c.scale.is_contiguous()):
            raise _lib.NvkError("Fp4Cache must be contiguous uint8 [num_blocks, Hkv, block_size, "
                                "D / 2] and float16 [num_blocks, Hkv, D / 32, block_size]")
    nb, hkv, bs, half = k_cache.data.shape
    if (k_cache.data.shape != v_cache.data.shape or half not in (32, 64) or bs % 16
            or k_cache.scale.shape != (nb, hkv, half // 16, bs)
            or v_cache.scale.shape != k_cache.scale.shape):
        raise _lib.NvkError("Fp4Cache shapes disagree, or head_dim is not 128 or 64, or block_size "
                            "not a multiple of 16")
    return nb, bs, hkv, 2 * half


def _rows_dtype(dtype: torch.dtype) -> int:
    if dtype == torch.bfloat16:
        return _lib.NVK_DTYPE_BF16
    if dtype == torch.float16:
        return _lib.NVK_DTYPE_F16
    raise _lib.NvkError(f"a 4-bit cache takes and gives bfloat16 and float16 rows, got {dtype}")


def fp4_store(key: torch.Tensor, value: torch.Tensor, k_cache: Fp4Cache, v_cache: Fp4Cache,
              slot_mapping: torch.Tensor) -> None:
    """``store_kvcache`` into 4-bit caches: the same arguments and checks; rows bf16 or f16, 16-byte
    aligned."""
    nb, bs, hkv, d = _check_caches(k_cache, v_cache)
    dtype = _rows_dtype(key.dtype)
    N = key.shape[0]
    assert key.shape == value.shape == (N, hkv, d) and key.dtype == value.dtype
    assert key.stride(-1) == 1 and value.stride(-1) == 1
    assert key.stride(1) == d and value.stride(1) == d
    assert slot_mapping.numel() == N
    dev = _lib.require_gpu(key, value, *k_cache, *v_cache, slot_mapping)
    slots = _lib.int32(slot_mapping)
    with _lib.on_device(dev):
        code = _lib.load().nvk_fp4_store(
            key.data_ptr(), key.stride(0), value.data_ptr(), value.stride(0),
            k_cache.data.data_ptr(), k_cache.scale.data_ptr(), v_cache.data.data_ptr(),
            v_cache.scale.data_ptr(), slots.data_ptr(), N, hkv, d, bs, nb, dtype,
            _lib.stream_ptr(dev))
    _lib.check(code)


def load_kvcache(k_cache: Fp4Cache, v_cache: Fp4Cache, slot_mapping: torch.Tensor,
                 dtype: torch.dtype = torch.bfloat16) -> tuple[torch.Tensor, torch.Tensor]:
    """The keys and values that 4-bit caches hold at the slots, [N, num_kv_heads, head_dim] of
    ``dtype`` (bfloat16 or float16) each: what ``store_kvcache`` with the same slots stored, as it
    was rounded.  A slot outside the cache (-1) gives zeros."""
    nb, bs, hkv, d = _check_caches(k_cache, v_cache)
    code = _rows_dtype(dtype)
    dev = _lib.require_gpu(*k_cache, *v_cache, slot_mapping)
    slots = _lib.int32(slot_mapping).view(-1)
    N = slots.numel()
    key, value = (torch.empty(N, hkv, d, dtype=dtype, device=dev) for _ in range(2))
    with _lib.on_device(dev):
        st = _lib.load().nvk_fp4_load(
            k_cache.data.data_ptr(), k_cache.scale.data_ptr(), v_cache.data.data_ptr(),
            v_cache.scale.data_ptr(), slots.data_ptr(), N, hkv, d, bs, nb, key.data_ptr(), hkv * d,
            value.data_ptr(), hkv * d, code, _lib.stream_ptr(dev))
    _lib.check(st)
    return key, value


def fp4_attention(q: torch.Tensor, k_cache: Fp4Cache, v_cache: Fp4Cache, seqlens_k: torch.Tensor,
                  block_table: torch.Tensor, softmax_scale=None, cu_seqlens_q=None,
                  max_seqlen_q: int = 1, max_seqlen_k: int | None = None,
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of q [tokens, Hq, D] over 4-bit caches.  Without ``cu_seqlens_q`` every
    sequence has ``max_seqlen_q`` queries and ``seqlens_k`` [B] keys; with it both are prefix sums
    [B + 1].  The queries are the last of their sequence's keys.  ``max_seqlen_k`` bounds the keys of
    a sequence (None: what the block table holds).  Returns [tokens, Hq, D] (or fills ``out``)."""
    nb, bs, hkv, d = _check_caches(k_cache, v_cache)
    dev = _lib.require_gpu(q, *k_cache, *v_cache, seqlens_k, block_table, cu_seqlens_q)
    dtype = _rows_dtype(q.dtype)
    if q.dim() != 3 or q.stride(-1) != 1 or q.shape[2] != d:
        raise _lib.NvkError("q must be [tokens, heads, head_dim] with unit last stride and the "
                            "caches' head_dim")
    tq, hq, _ = q.shape
    lens, bt = _lib.int32(seqlens_k), _lib.int32(block_table)
    cu_q = None if cu_seqlens_q is None else _lib.int32(cu_seqlens_q)
    batch = lens.numel() - (cu_q is not None)
    if cu_q is not None and cu_q.numel() != lens.numel():
        raise _lib.NvkError("cu_seqlens_q and cu_seqlens_k disagree on the batch size")
    if cu_q is None and batch * max_seqlen_q != tq:
        raise _lib.NvkError("q and cache_seqlens disagree on the batch size")
    if bt.dim() != 2 or bt.shape[0] != batch:
        raise _lib.NvkError("block_table must be [batch, max_blocks]")
    if out is None:
        out = torch.empty((tq, hq, d), dtype=q.dtype, device=dev)
    elif out.shape != q.shape or out.dtype != q.dtype or out.device != dev or out.stride(-1) != 1:
        raise _lib.NvkError("out must be like q, with unit last stride")
    scale = float(softmax_scale) if softmax_scale is not None else d ** -0.5
    lib = _lib.load()
    mq, mk, width = int(max_seqlen_q), int(max_seqlen_k or 0), bt.shape[1]
    ws_bytes = lib.nvk_fp4_attention_workspace_size(batch, mq, mk, hq, hkv, d, bs, width)
    ws = _lib.workspace(dev, ws_bytes)
    with _lib.on_device(dev):
        code = lib.nvk_fp4_attention(
            q.data_ptr(), q.stride(0), q.stride(1), tq, k_cache.data.data_ptr(),
            k_cache.scale.data_ptr(), v_cache.data.data_ptr(), v_cache.scale.data_ptr(),
            _lib.ptr(cu_q), lens.data_ptr(), batch, mq, mk, bt.data_ptr(), bt.stride(0), width, bs,
            nb, hq, hkv, d, scale, out.data_ptr(), out.stride(0), out.stride(1), _lib.ptr(ws),
            ws_bytes, dtype, _lib.stream_ptr(dev))
    _lib.check(code)
    return out
