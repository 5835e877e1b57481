"""Q/K head RMSNorm, RoPE and in-place KV-cache update on B200.

Drop-in for engine/kernels/qk_rope.py:87-129 (same signature, asserts and return value):
one launch of fb_qk_norm_rope_append writes token-major Q and appends K (normed, rotated)
and V (copied) at each token's cache slot. ``qk_rope_cache_q8`` is the same call on an 8-bit
cache (kernels.quant.QuantCache; fb_qk_norm_rope_append_q8, no counterpart in the reference).
"""

import torch

from kernels import _native
from kernels._native import check, lib, ptr, stream
from kernels.merged import Split, source


def qk_rope_cache(packed, q_norm, k_norm, cos, sin, position, keys, values, q_heads, prefill=False, rows=False, phases=None):
    """BF16 packed QKV and [B,Hkv,C,D] caches, for prefill or one decode token.

    Native BF16 phases [1,T,D] are shared by batch rows. Prefill writes [0,T); decode
    writes T slots starting at the device-side scalar position (per row with ``rows``).
    Return a [B,Hq,T,D] view of token-major Q storage (contiguous when T is one).
    """
    batch, kv_heads, capacity, dim = keys.shape
    split = isinstance(packed, Split)
    packed, splits, count, shape = source(packed)
    tokens = shape[1]
    assert keys.dtype == values.dtype == torch.bfloat16
    assert packed.dtype == (torch.float32 if split else torch.bfloat16)
    assert packed.is_contiguous() and keys.is_contiguous() and values.is_contiguous()
    assert shape == (batch, tokens, (q_heads + 2 * kv_heads) * dim)
    assert 0 < tokens <= capacity
    assert values.shape == keys.shape and dim % 2 == 0
    assert not (rows and prefill)
    table = phases is not None
    if table:
        assert rows and phases.shape == (batch, tokens) and phases.is_contiguous() and phases.dtype == torch.int64
        assert cos.shape == sin.shape and cos.shape[-1] == dim and cos.numel() // dim >= capacity
    else:
        assert cos.numel() == sin.numel() == (batch if rows else 1) * tokens * dim
    assert cos.is_contiguous() and sin.is_contiguous()
    assert position.shape == ((tokens,) if prefill else (batch,) if rows else (1,))
    assert position.dtype == torch.int64
    _native.require_cuda(packed, keys, values, cos, sin, position)
    query = torch.empty((batch, tokens, q_heads, dim), device=packed.device, dtype=keys.dtype)
    mode = 1 if prefill else 2 if rows else 0
    check(lib.fb_qk_norm_rope_append(
        ptr(packed), splits if packed.dtype == torch.float32 else 0, ptr(q_norm.weight), ptr(k_norm.weight),
        float(q_norm.variance_epsilon), float(k_norm.variance_epsilon), ptr(cos), ptr(sin),
        ptr(position), ptr(phases) if table else None, ptr(query), ptr(keys), ptr(values),
        batch, tokens, q_heads, kv_heads, dim, capacity, mode, 1 if table else 0, stream(),
    ), "fb_qk_norm_rope_append")
    return query.transpose(1, 2)


def qk_rope_cache_q8(packed, q_norm, k_norm, cos, sin, position, cache, q_heads, prefill=False, rows=False, phases=None,
                     table=False):
    """``qk_rope_cache`` into a ``QuantCache``: norm and RoPE in fp32, Q rounded once to BF16, K and V
    once to e4m3 under their block's scale. ``table`` (decode mode) or ``phases`` (rows mode): cos
    and sin are whole tables of at least ``cache.capacity`` rows, read at the device-side position.
    Rows at a negative position get nothing appended."""
    split = isinstance(packed, Split)
    data, splits = (packed.partial, packed.splits) if split else (packed, 0)
    batch, kv_heads, capacity, dim, device = cache.batch, cache.kv_heads, cache.capacity, cache.dim, cache.device
    shape = packed.shape
    tokens = shape[1]
    assert data.dtype == (torch.float32 if split else torch.bfloat16) and data.is_contiguous()
    assert shape == (batch, tokens, (q_heads + 2 * kv_heads) * dim) and q_heads > 0
    assert not split or splits > 0 and data.shape == (splits, batch * tokens, shape[2])
    assert 0 < tokens <= capacity
    assert not (rows and prefill) and not (table and (rows or prefill))
    if phases is not None:
        assert rows and phases.shape == (batch, tokens) and phases.is_contiguous() and phases.dtype == torch.int64
    whole = table or phases is not None
    assert cos.dtype == sin.dtype == torch.bfloat16 and cos.is_contiguous() and sin.is_contiguous()
    if whole:
        assert cos.shape == sin.shape and cos.shape[-1] == dim and cos.numel() >= capacity * dim
    else:
        assert cos.numel() == sin.numel() == (batch if rows else 1) * tokens * dim
    assert position.shape == ((tokens,) if prefill else (batch,) if rows else (1,))
    assert position.dtype == torch.int64 and position.is_contiguous()
    q_weight, k_weight = q_norm.weight, k_norm.weight
    assert q_weight.dtype == k_weight.dtype == torch.bfloat16 and q_weight.numel() == k_weight.numel() == dim
    assert q_weight.is_contiguous() and k_weight.is_contiguous()
    if not (data.get_device() == cos.get_device() == sin.get_device() == position.get_device() ==
            q_weight.get_device() == k_weight.get_device() == device.index) or phases is not None:
        _native.require_device(device, data, cos, sin, position, phases, q_weight, k_weight)
    token = q_heads * dim  # token-major, seen as [B, Hq, T, D]
    query = cos.new_empty_strided((batch, q_heads, tokens, dim), (tokens * token, dim, token, 1))
    _native.launch(
        "fb_qk_norm_rope_append_q8", device, data.data_ptr(), splits, q_weight.data_ptr(), k_weight.data_ptr(),
        q_norm.variance_epsilon, k_norm.variance_epsilon, cos.data_ptr(), sin.data_ptr(), position.data_ptr(),
        None if phases is None else phases.data_ptr(), query.data_ptr(), cache.address, tokens, q_heads,
        1 if prefill else 2 if rows else 0, 1 if whole else 0)
    return query
