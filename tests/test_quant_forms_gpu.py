"""The forms of the 8-bit attention one by one: each test asserts which form its shape takes (a cluster per
unit needs no workspace; a grid of slices does), with 64-bit restatements as in test_quant_gpu.py."""

import math

import pytest
import torch

from oracle import quant as oq

pytestmark = pytest.mark.gpu
DEV = "cuda"
#: A capacity from which more units than SMs are cut into slices of a persistent grid.
LONG = 4800


@pytest.fixture(autouse=True)
def _no_device_errors():
    from kernels import _native
    _native.device_error()
    yield
    assert _native.device_error() == 0, "a kernel raised its device error word"


def handle(cache, device=DEV):
    from kernels.quant import QuantCache
    c = oq.to_device(cache, device)
    return QuantCache(c["keys"], c["values"], c["key_scales"], c["value_scales"], c["block"])


def check(out, expect, bound):
    out = out.cpu().double()
    assert torch.isfinite(out).all()
    off = (out - expect).abs()
    assert (off <= bound).all(), f"off by {float((off / bound.clamp_min(1e-300)).max())} bounds"


@pytest.mark.parametrize("sliced", [False, True])
@pytest.mark.parametrize("tokens,groups,dim", [(1, 4, 128), (1, 7, 64), (3, 4, 128), (5, 4, 64), (7, 4, 128)])
def test_small_weights_beside_a_leader(sliced, tokens, groups, dim):
    """One slot leads every other by 25.3 in log2 and its value is zero (an attention sink): the output is what
    the others' weights of 2^-25.3 make of their values, all of one sign. Weights that small must not vanish in
    the value product while the denominator counts them."""
    from kernels.decode_attention import block_attention_q8, decode_attention_q8
    g = torch.Generator().manual_seed(tokens + groups + dim)
    batch, kv_heads, capacity = (20, 8, LONG) if sliced else (2, 2, 700)
    cache = oq.random_cache(batch, kv_heads, capacity, dim, 64, g)
    cache["values"] = cache["values"].float().abs().clamp_min(16).to(oq.E4M3)
    keys = cache["keys"].float()
    keys[..., 0] = 0
    position = torch.randint(500, 690 - tokens, (batch,), generator=g)
    values = cache["values"].float()
    for b in range(batch):
        leader = int(torch.randint(0, int(position[b]) + 1, (1,), generator=g))
        keys[b, :, leader, 0] = 448.0
        values[b, :, leader] = 0
    cache["keys"], cache["values"] = keys.to(oq.E4M3), values.to(oq.E4M3)
    cache["key_scales"] = torch.full_like(cache["key_scales"], 2.0 ** -6)
    query = 0.002 * torch.randn(batch, tokens, kv_heads * groups, dim, generator=g)
    query[..., 0] = 1.0
    query, scale = query.bfloat16(), 25.3 * math.log(2) / 7
    chain = torch.full((batch,), tokens)
    expect, bound = oq.attention(query, cache, position, scale, None if tokens == 1 else chain)
    assert (bound < 0.1 * expect).all()  # nothing vanishes within the bound
    c = handle(cache)
    assert (c.workspace_bytes(tokens, kv_heads * groups) > 0) == sliced
    if tokens == 1:
        out = decode_attention_q8(query.transpose(1, 2).contiguous().to(DEV), c, position.to(DEV), scale)
    else:
        out = block_attention_q8(query.to(DEV), c, position.to(DEV), scale, chain.to(DEV))
    check(out, expect, bound)


@pytest.mark.parametrize("batch,kv_heads,capacity,tokens,q_heads,sliced", [
    (64, 8, 2048, 1, 16, False), (64, 8, 32768, 1, 16, True), (8, 8, 32768, 5, 32, False), (20, 8, LONG, 1, 32, True),
    (1, 2, 64, 1, 16, False)])
def test_workspace_says_which_form(batch, kv_heads, capacity, tokens, q_heads, sliced):
    """Units of short rows, and up to one a SM, run as clusters without a workspace; the others take partials of
    two CTAs an SM."""
    import ctypes
    from kernels._native import Q8Cache, lib
    c = Q8Cache(1 << 20, 1 << 20, 1 << 20, 1 << 20, batch, kv_heads, capacity, 128, 64)  # sizes only
    need = lib.fb_attention_q8_workspace(ctypes.byref(c), tokens, q_heads)
    slots = 2 * torch.cuda.get_device_properties(0).multi_processor_count + batch * kv_heads
    width = tokens * (q_heads // kv_heads)
    assert need == (-(-slots * width * 128 * 4 // 256) * 256 + slots * width * 16 if sliced else 0)
