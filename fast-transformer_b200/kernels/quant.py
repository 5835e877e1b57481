"""Quantised operands of the decode step on B200: an 8-bit KV cache and 4-bit projection weights.

``QuantCache`` is one layer's cache as e4m3 codes with an fp32 scale per (row, KV head, block of
slots). ``kernels.qk_rope.qk_rope_cache_q8`` appends to it, ``kernels.decode_attention``'s
``decode_attention_q8`` and ``block_attention_q8`` attend over it, ``kernels.spec.relocate_q8`` moves
a slot. ``Weight4`` is a projection's weights as 4-bit codes with a bf16 scale per row and group of
columns, laid out once for ``kernels.linear.linear`` and ``swiglu_linear``, which take it in
place of a tensor. The reference has neither: its cache and weights are bf16.
"""

import ctypes

import torch

from kernels import _native
from kernels._native import lib

#: Slots that share a scale.
BLOCKS = (16, 32, 64)
#: Weight columns that share a scale.
GROUPS = (32, 64, 128)
CODE = torch.float8_e4m3fn


class QuantCache:
    """One layer's 8-bit cache: ``keys`` and ``values`` [B, Hkv, C, D] e4m3 codes, ``key_scales`` and
    ``value_scales`` fp32 [B, Hkv, ceil(C / block)], all contiguous on one CUDA device. Slot c of
    a head stands for ``codes[c] * scales[c // block]``. Built on existing tensors, which it keeps
    and the append updates in place."""

    __slots__ = ("_keys", "_values", "_key_scales", "_value_scales", "block", "batch", "kv_heads", "capacity", "dim",
                 "device", "_struct", "address", "_workspace")

    def __init__(self, keys, values, key_scales, value_scales, block=64):
        assert block in BLOCKS
        assert keys.dtype == values.dtype == CODE and keys.dim() == 4 and values.shape == keys.shape
        batch, kv_heads, capacity, dim = keys.shape
        assert batch > 0 and kv_heads > 0 and capacity > 0 and dim in (64, 128)
        scales = (batch, kv_heads, -(-capacity // block))
        assert key_scales.dtype == value_scales.dtype == torch.float32
        assert key_scales.shape == scales and value_scales.shape == scales
        for t in (keys, values, key_scales, value_scales):
            assert t.is_contiguous()
        _native.require_device(keys.device, keys, values, key_scales, value_scales)
        assert keys.data_ptr() % 16 == 0 and values.data_ptr() % 16 == 0
        self._keys, self._values = keys, values
        self._key_scales, self._value_scales = key_scales, value_scales
        self.block, self.device = block, keys.device
        self.batch, self.kv_heads, self.capacity, self.dim = batch, kv_heads, capacity, dim
        self._struct = _native.Q8Cache(keys.data_ptr(), values.data_ptr(), key_scales.data_ptr(),
                                       value_scales.data_ptr(), batch, kv_heads, capacity, dim, block)
        self.address = ctypes.addressof(self._struct)  # fb_q8_cache*
        self._workspace = {}

    @classmethod
    def zeros(cls, batch, kv_heads, capacity, dim, block=64, device="cuda"):
        """An empty cache of its own buffers."""
        def codes():
            return torch.zeros((batch, kv_heads, capacity, dim), dtype=torch.uint8, device=device).view(CODE)

        def scales():
            return torch.zeros((batch, kv_heads, -(-capacity // block)), dtype=torch.float32, device=device)

        return cls(codes(), codes(), scales(), scales(), block)

    keys = property(lambda self: self._keys)
    values = property(lambda self: self._values)
    key_scales = property(lambda self: self._key_scales)
    value_scales = property(lambda self: self._value_scales)

    def dequantized(self):
        """(keys, values) as fp32 tensors of what the codes stand for (torch; for inspection)."""
        def expand(codes, scales):
            return codes.float() * scales.repeat_interleave(self.block, 2)[:, :, :self.capacity, None]

        return expand(self._keys, self._key_scales), expand(self._values, self._value_scales)

    def workspace_bytes(self, tokens, q_heads):
        """Bytes an attention call of this shape needs (0: none; fixed per shape and device)."""
        key = (tokens, q_heads)
        need = self._workspace.get(key)
        if need is None:
            with torch.cuda.device(self.device):
                need = int(lib.fb_attention_q8_workspace(self.address, tokens, q_heads))
            if need == ctypes.c_size_t(-1).value:
                raise ValueError(f"8-bit attention of {tokens} x {q_heads} queries over a cache of {self.batch} x "
                                 f"{self.kv_heads} x {self.capacity} slots is not supported, or {self.device} refuses "
                                 "its kernels")
            self._workspace[key] = need
        return need


class Weight4:
    """A projection's [N, K] weights in 4 bits: ``packed`` holds the codes and one bf16 scale per row and
    ``group`` columns in the kernel's layout. Made by ``pack_weight4`` or ``quantize_weight4``."""

    __slots__ = ("packed", "shape", "n", "k", "group", "device")

    def __init__(self, packed, shape, group):
        self.packed = packed
        self.shape, self.group, self.device = torch.Size(shape), group, packed.device
        self.n, self.k = self.shape

    @property
    def nbytes(self):
        """Bytes one product reads of it."""
        return self.packed.numel()

    def dequantized(self):
        """bf16 [N, K]: code * scale, rounded once (fb_w4_dequantize)."""
        n, k = self.shape
        out = torch.empty((n, k), dtype=torch.bfloat16, device=self.device)
        _native.launch("fb_w4_dequantize", self.device, self.packed.data_ptr(), out.data_ptr(), n, k, self.group)
        return out


def _check_shape(n, k, group):
    if group not in GROUPS:
        raise ValueError(f"4-bit weights take groups of {GROUPS} columns, not {group}")
    if n <= 0 or k <= 0 or n % 8 or k % group:
        raise ValueError(f"4-bit weights [{n}, {k}] need rows in multiples of 8 and columns in multiples of {group}")


def pack_weight4(codes, scales):
    """``Weight4`` of int8 codes [N, K] in -8..7 and bf16 scales [N, K / group] (weights are laid out
    once, at load: the call checks codes and scales on the host and so synchronises)."""
    if codes.dtype != torch.int8 or scales.dtype != torch.bfloat16 or codes.dim() != 2 or scales.dim() != 2:
        raise ValueError("4-bit weights are packed from int8 codes [N, K] and bf16 scales [N, K / group]")
    n, k = codes.shape
    if scales.shape[0] != n or scales.shape[1] == 0 or k % scales.shape[1]:
        raise ValueError(f"scales {tuple(scales.shape)} do not group the columns of {tuple(codes.shape)}")
    group = k // scales.shape[1]
    _check_shape(n, k, group)
    _native.require_device(codes.device, codes, scales)
    low, high, finite = torch.stack((*torch.aminmax(codes), torch.isfinite(scales).all().to(torch.int8))).tolist()
    if low < -8 or high > 7:
        raise ValueError("4-bit codes lie in -8..7")
    if not finite:  # a product scales its groups' sums: 0 times infinity would not show
        raise ValueError("4-bit weights take finite scales")
    codes, scales = codes.contiguous(), scales.contiguous()
    packed = torch.empty(int(lib.fb_w4_packed_bytes(n, k, group)), dtype=torch.uint8, device=codes.device)
    _native.launch("fb_w4_pack", codes.device, codes.data_ptr(), scales.data_ptr(), packed.data_ptr(), n, k, group)
    # a product may read its weights before the kernel ahead of it ends: that must not be this one
    torch.cuda.current_stream(codes.device).synchronize()
    return Weight4(packed, (n, k), group)


def quantize_weight4(weight, group=128):
    """``Weight4`` nearest to a [N, K] tensor: per row and group the scale that maps the largest
    magnitude to 7 (rounded to bf16), codes rounded to nearest even."""
    if weight.dim() != 2 or not weight.is_floating_point():
        raise ValueError("quantize_weight4 takes a floating-point [N, K] tensor")
    n, k = weight.shape
    _check_shape(n, k, group)
    _native.require_device(weight.device, weight)
    parts = weight.float().reshape(n, k // group, group)
    scales = (parts.abs().amax(-1) / 7.0).to(torch.bfloat16)
    if not bool(torch.isfinite(scales).all()):
        raise ValueError("quantize_weight4 takes finite weights")
    divisor = torch.where(scales == 0, torch.ones_like(scales), scales).float()
    codes = (parts / divisor[..., None]).round().clamp_(-8, 7).to(torch.int8).reshape(n, k)
    return pack_weight4(codes, scales)
