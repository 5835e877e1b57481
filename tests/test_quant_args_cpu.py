"""Sizes and refusals of the quantised decode operators that need no GPU."""

import ctypes

import pytest
import torch

p = ctypes.c_void_p(1 << 20)  # never dereferenced
NULL = None
NO_DEVICE = not torch.cuda.is_available()


def cache(batch=1, kv_heads=2, capacity=64, dim=128, block=64):
    from kernels._native import Q8Cache
    return Q8Cache(1 << 20, 1 << 20, 1 << 20, 1 << 20, batch, kv_heads, capacity, dim, block)


def test_misaligned_pointers_are_refused():
    """Codes can lie at any byte; the kernels read and write them (and what they expand to) in wider words."""
    from kernels._native import lib

    def at(offset):
        return ctypes.c_void_p((1 << 20) + offset)

    for offset in (1, 2, 3):
        assert lib.fb_spec_relocate_q8(at(offset), p, 4, 2, 2, 64, 128, 64, p, p, NULL) == -1
    for offset in (1, 2, 4, 8):
        assert lib.fb_w4_pack(p, p, at(offset), 8, 32, 32, NULL) == -1
        assert lib.fb_w4_dequantize(at(offset), p, 8, 32, 32, NULL) == -1
        assert lib.fb_w4_dequantize(p, at(offset), 8, 32, 32, NULL) == -1


@pytest.mark.skipif(not NO_DEVICE, reason="sizes of a host without a device")
@pytest.mark.parametrize("batch,kv_heads,q_heads,tokens,dim", [(1, 2, 16, 1, 128), (64, 8, 16, 1, 128), (3, 2, 14, 5, 64),
                                                              (2, 1, 36, 1, 64)])
def test_attention_workspace_without_a_device(batch, kv_heads, q_heads, tokens, dim):
    """The most any form takes: fp32 partials and four statistics for each of 296 CTAs and each unit."""
    from kernels._native import lib
    members = tokens * (q_heads // kv_heads)
    chunks = -(-members // 32)
    width = -(-members // chunks)
    slots = 2 * 148 + batch * kv_heads * chunks
    acc = -(-slots * width * dim * 4 // 256) * 256
    c = cache(batch, kv_heads, 2048, dim)
    assert lib.fb_attention_q8_workspace(ctypes.byref(c), tokens, q_heads) == acc + slots * width * 16


def test_weights_past_the_layouts_index_range_are_refused():
    """The layout's kernels count rows of codes in 32 bits: at most 2^34 weights."""
    from kernels._native import lib
    assert lib.fb_w4_packed_bytes(1 << 20, 1 << 14, 128) == (1 << 33) + (1 << 20) * (1 << 7) * 2
    for n, k in ((1 << 20, (1 << 14) + 128), (1 << 22, 1 << 14), (1 << 22, 1 << 20)):
        assert lib.fb_w4_packed_bytes(n, k, 128) == 0
        assert lib.fb_w4_pack(p, p, p, n, k, 128, NULL) == -2
        assert lib.fb_w4_dequantize(p, p, n, k, 128, NULL) == -2
        assert lib.fb_linear_w4(p, p, p, 1, n, k, 128, 0, NULL) == -2


@pytest.mark.parametrize("partial", [(0, 3, 1024), (2, 2, 1024), (2, 3, 1023), (3, 1024)])
def test_append_refuses_partials_that_are_not_its_shape(partial):
    """A Split carries its logical shape beside its buffer: the two have to agree before a kernel reads by the
    first."""
    from types import SimpleNamespace
    from kernels.merged import Split
    from kernels.qk_rope import qk_rope_cache_q8
    c = SimpleNamespace(batch=3, kv_heads=2, capacity=40, dim=128, device=torch.device("cuda", 0), block=16)
    norm = SimpleNamespace(weight=torch.ones(128, dtype=torch.bfloat16), variance_epsilon=1e-6)
    phase = torch.zeros(1, 1, 128, dtype=torch.bfloat16)
    with pytest.raises(AssertionError):
        qk_rope_cache_q8(Split(torch.zeros(partial), (3, 1, 1024)), norm, norm, phase, phase,
                         torch.zeros(1, dtype=torch.int64), c, 4)
