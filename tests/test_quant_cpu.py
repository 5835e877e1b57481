"""Refusals of the quantised decode operators, on the CPU: the C entry points check their arguments
before anything is launched, the wrappers before they call."""

import ctypes

import pytest
import torch

p = ctypes.c_void_p(1 << 20)  # never dereferenced
NULL = None


def test_append_refusals():
    from kernels._native import lib

    def call(packed=p, splits=0, keys=p, batch=1, tokens=1, q_heads=4, kv_heads=2, dim=128, capacity=64, block=64,
             mode=0, table=0, phases=NULL):
        return lib.fb_qk_norm_rope_append_q8(packed, splits, p, p, 1e-6, 1e-6, p, p, p, phases, p, keys, p, p, p, batch,
                                             tokens, q_heads, kv_heads, dim, capacity, block, mode, table, NULL)

    assert call(packed=NULL) == -1 and call(keys=NULL) == -1
    assert call(batch=0) == -1 and call(tokens=0) == -1 and call(kv_heads=0) == -1 and call(splits=-1) == -1
    assert call(mode=3) == -1 and call(mode=1, table=1) == -1 and call(phases=p, mode=2) == -1
    assert call(dim=96) == -2 and call(block=48) == -2 and call(block=128) == -2 and call(tokens=65) == -2


def test_relocate_refusals():
    from kernels._native import lib
    assert lib.fb_spec_relocate_q8(NULL, p, 4, 2, 2, 64, 128, 64, p, p, NULL) == -1
    assert lib.fb_spec_relocate_q8(p, p, 0, 2, 2, 64, 128, 64, p, p, NULL) == -1
    assert lib.fb_spec_relocate_q8(p, p, 4, 2, 2, 64, 60, 64, p, p, NULL) == -2
    assert lib.fb_spec_relocate_q8(p, p, 4, 2, 2, 64, 64, 8, p, p, NULL) == -2


def test_attention_refusals():
    from kernels._native import lib
    need = lib.fb_attention_q8_workspace(4, 1, 16, 8, 128, 2048, 64)
    assert need > 0

    def call(q=p, per_row=1, chain=NULL, nbytes=need, batch=4, tokens=1, q_heads=16, kv_heads=8, dim=128,
             capacity=2048, block=64, workspace=p):
        return lib.fb_attention_q8(q, p, p, p, p, p, per_row, chain, p, workspace, nbytes, batch, tokens, q_heads,
                                   kv_heads, dim, capacity, block, 0.1, NULL)

    assert call(q=NULL) == -1 and call(workspace=NULL) == -1 and call(batch=0) == -1
    assert call(tokens=2) == -1                       # several tokens need a chain
    assert call(chain=p, per_row=0) == -1             # a block's positions are per row
    assert call(dim=96) == -2 and call(block=24) == -2 and call(q_heads=15) == -2 and call(batch=1025) == -2
    assert call(kv_heads=8, q_heads=8, batch=1024, capacity=1 << 20) == -2   # 2^33 cache rows
    assert call(tokens=2049, chain=p) == -2           # more tokens than slots
    assert call(nbytes=need - 1) == -5
    assert call(q=ctypes.c_void_p((1 << 20) + 2)) == -1 and call(workspace=ctypes.c_void_p((1 << 20) + 8)) == -1
    assert lib.fb_attention_q8_workspace(4, 1, 16, 8, 96, 2048, 64) == 0


def test_linear_refusals():
    from kernels._native import lib

    def call(x=p, m=4, n=128, k=128, group=64, epilogue=0):
        return lib.fb_linear_w4(x, p, p, p, m, n, k, group, epilogue, NULL)

    assert call(x=NULL) == -1 and call(m=0) == -1 and call(epilogue=3) == -1
    assert call(m=65) == -2 and call(n=12) == -2 and call(k=96) == -2 and call(group=16) == -2 and call(n=0) == -2
    assert call(n=72, epilogue=2) == -2
    assert call(x=ctypes.c_void_p((1 << 20) + 8)) == -1
    assert lib.fb_w4_packed_bytes(100, 64, 32) == 0 and lib.fb_w4_scale_bytes(104, 48, 32) == 0
    # tiles of 16 rows and 64 columns, padded
    assert lib.fb_w4_packed_bytes(24, 96, 32) == 2 * 2 * 512 and lib.fb_w4_scale_bytes(24, 96, 32) == 2 * 4 * 32
    assert lib.fb_w4_pack(NULL, p, p, p, 8, 32, 32, NULL) == -1 and lib.fb_w4_pack(p, p, p, p, 8, 32, 16, NULL) == -2
    assert lib.fb_w4_dequantize(p, NULL, p, 8, 32, 32, NULL) == -1


def test_wrappers_refuse():
    from kernels.quant import QuantCache, pack_weight4, quantize_weight4
    from kernels.spec import relocate_q8

    def parts(batch=1, heads=2, capacity=40, dim=64, block=16):
        codes = torch.zeros(batch, heads, capacity, dim, dtype=torch.uint8).view(torch.float8_e4m3fn)
        return codes, codes.clone(), torch.zeros(batch, heads, 3), torch.zeros(batch, heads, 3)

    k, v, ks, vs = parts()
    with pytest.raises(ValueError):
        QuantCache(k, v, ks, vs, 16)  # CPU tensors
    for bad in ((k, v, ks, vs, 8), (k.float(), v, ks, vs, 16), (k, v, ks[..., :2], vs, 16), (k, v[:, :1], ks, vs, 16),
                (k, v, ks.double(), vs, 16), (k.transpose(0, 1), v.transpose(0, 1), ks, vs, 16), (k, v, ks, vs, 64)):
        with pytest.raises(AssertionError):
            QuantCache(*bad)
    codes = torch.zeros(16, 64, dtype=torch.int8)
    scales = torch.ones(16, 2, dtype=torch.bfloat16)
    for bad in ((codes, scales), (codes.short(), scales), (codes, scales.float()), (codes, scales[:8]),
                (codes[:12], scales[:12]), (codes, torch.ones(16, 1, dtype=torch.bfloat16)[:, :0]),
                (codes, torch.ones(16, 4, dtype=torch.bfloat16))):
        with pytest.raises(ValueError):
            pack_weight4(*bad)
    with pytest.raises(ValueError):
        quantize_weight4(torch.zeros(16, 64), 48)
    with pytest.raises(ValueError):
        quantize_weight4(torch.zeros(16, 64, dtype=torch.int32), 64)
    store = torch.zeros(2, 1, 1, 1, 16, 64, dtype=torch.uint8).view(torch.float8_e4m3fn)
    moves = torch.zeros(1, dtype=torch.int64)
    with pytest.raises(ValueError):
        relocate_q8(store, torch.zeros(2, 1, 1, 1, 1), 16, moves, moves)  # CPU
    with pytest.raises(AssertionError):
        relocate_q8(store, torch.zeros(2, 1, 1, 1, 2), 16, moves, moves)
