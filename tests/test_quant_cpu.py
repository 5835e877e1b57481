"""Refusals of the quantised decode operators, on the CPU: the C entry points check their arguments
before anything is launched, the wrappers before they call."""

import ctypes

import pytest
import torch

p = ctypes.c_void_p(1 << 20)  # never dereferenced
NULL = None


def cache(batch=1, kv_heads=2, capacity=64, dim=128, block=64, keys=1 << 20):
    from kernels._native import Q8Cache
    return Q8Cache(keys, 1 << 20, 1 << 20, 1 << 20, batch, kv_heads, capacity, dim, block)


def test_append_refusals():
    from kernels._native import lib

    def call(packed=p, splits=0, tokens=1, q_heads=4, mode=0, table=0, phases=NULL, **sizes):
        c = cache(**sizes)
        return lib.fb_qk_norm_rope_append_q8(packed, splits, p, p, 1e-6, 1e-6, p, p, p, phases, p, ctypes.byref(c), tokens,
                                             q_heads, mode, table, NULL)

    assert call(packed=NULL) == -1 and call(keys=None) == -1
    assert lib.fb_qk_norm_rope_append_q8(p, 0, p, p, 1e-6, 1e-6, p, p, p, NULL, p, NULL, 1, 4, 0, 0, NULL) == -1
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
    bad = ctypes.c_size_t(-1).value

    def need(tokens=1, q_heads=16, **sizes):
        return lib.fb_attention_q8_workspace(ctypes.byref(cache(**{**shape, **sizes})), tokens, q_heads)

    shape = dict(batch=64, kv_heads=8, capacity=2048, dim=128, block=64)
    assert 0 < need() < bad  # more units than the machine holds clusters: the persistent form
    assert need(dim=96) == bad and need(q_heads=15) == bad and need(batch=1025) == bad and need(tokens=2049) == bad

    def call(q=p, per_row=1, chain=NULL, nbytes=None, workspace=p, tokens=1, q_heads=16, **sizes):
        c = cache(**{**shape, **sizes})
        return lib.fb_attention_q8(q, ctypes.byref(c), p, per_row, chain, p, workspace, need() if nbytes is None else nbytes,
                                   tokens, q_heads, 0.1, NULL)

    assert call(q=NULL) == -1 and call(keys=None) == -1 and call(batch=0) == -1
    assert call(tokens=2) == -1                       # several tokens need a chain
    assert call(chain=p, per_row=0) == -1             # a block's positions are per row
    assert call(dim=96) == -2 and call(block=24) == -2 and call(q_heads=15) == -2 and call(batch=1025) == -2
    assert call(q_heads=8, batch=1024, capacity=1 << 20) == -2   # 2^33 cache rows
    assert call(tokens=2049, chain=p) == -2           # more tokens than slots
    assert call(q=ctypes.c_void_p((1 << 20) + 2)) == -1


def test_linear_refusals():
    from kernels._native import lib

    def call(x=p, m=4, n=128, k=128, group=64, epilogue=0):
        return lib.fb_linear_w4(x, p, p, m, n, k, group, epilogue, NULL)

    assert call(x=NULL) == -1 and call(m=0) == -1 and call(epilogue=3) == -1
    assert call(m=65) == -2 and call(n=12) == -2 and call(k=96) == -2 and call(group=16) == -2 and call(n=0) == -2
    assert call(n=72, epilogue=2) == -2
    assert call(x=ctypes.c_void_p((1 << 20) + 8)) == -1
    assert lib.fb_w4_packed_bytes(100, 64, 32) == 0 and lib.fb_w4_packed_bytes(104, 48, 32) == 0
    # tiles of 128 rows: half a byte a code, two bytes a scale
    assert lib.fb_w4_packed_bytes(24, 96, 32) == 128 * (48 + 3 * 2)
    assert lib.fb_w4_packed_bytes(136, 640, 128) == 256 * (320 + 5 * 2)
    assert lib.fb_w4_pack(NULL, p, p, 8, 32, 32, NULL) == -1 and lib.fb_w4_pack(p, p, p, 8, 32, 16, NULL) == -2
    assert lib.fb_w4_dequantize(p, NULL, 8, 32, 32, NULL) == -1


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
