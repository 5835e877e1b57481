"""The quantised decode operators on B200 against their 64-bit restatements (oracle/quant.py), whose
bounds count each rounding: attention over the 8-bit cache, the append, the slot move, 4-bit
projections."""

import math
from types import SimpleNamespace

import pytest
import torch

from oracle import quant as oq

pytestmark = pytest.mark.gpu
DEV = "cuda"
EPS = 1e-6


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


def poison(cache, position, tokens=1):
    """NaN codes in every slot behind each row's last token, as a reused cache may hold."""
    batch, capacity = cache["keys"].shape[0], cache["keys"].shape[2]
    for b in range(batch):
        p = int(position[b if len(position) > 1 else 0])
        end = 0 if p < 0 else min(p + tokens, capacity)
        for name in ("keys", "values"):
            cache[name].view(torch.uint8)[b, :, end:] = 0x7f
            whole = -(-end // cache["block"])
            cache[name[:-1] + "_scales"][b, :, whole:] = float("nan")


def check_attention(out, expect, bound):
    out = out.cpu().double()
    assert torch.isfinite(out).all()
    off = (out - expect).abs()
    assert (off <= bound).all(), f"off by {float((off / bound.clamp_min(1e-300)).max())} bounds"


# ------------------------------------------------------------------------------ attention
@pytest.mark.parametrize("batch,q_heads,kv_heads,dim,capacity,block,lengths", [
    (1, 16, 8, 128, 300, 64, [300]),
    (1, 1, 1, 64, 1, 16, [1]),
    (2, 8, 8, 128, 16, 16, [15, 16]),
    (4, 4, 1, 128, 777, 32, [1, 127, 128, 129]),
    (3, 14, 2, 64, 1003, 16, [0, 1003, 500]),
    (2, 16, 2, 128, 260, 64, [0, 0]),
    (2, 40, 2, 128, 200, 64, [200, 3]),       # 20 query heads a KV head: three column groups
    (2, 36, 1, 64, 150, 32, [150, 77]),       # 36: two member groups
    (5, 12, 4, 128, 2050, 64, [2050, 1, 0, 1999, 640]),
])
def test_decode_attention(batch, q_heads, kv_heads, dim, capacity, block, lengths):
    from kernels.decode_attention import decode_attention_q8
    g = torch.Generator().manual_seed(capacity + q_heads)
    cache = oq.random_cache(batch, kv_heads, capacity, dim, block, g)
    position = torch.tensor(lengths) - 1
    poison(cache, position)
    query = torch.randn(batch, q_heads, 1, dim, generator=g).bfloat16()
    expect, bound = oq.attention(query.transpose(1, 2), cache, position, 1 / math.sqrt(dim))
    c = handle(cache)
    out = decode_attention_q8(query.to(DEV), c, position.to(DEV), 1 / math.sqrt(dim))
    assert out.shape == (batch, 1, q_heads, dim) and out.dtype == torch.bfloat16
    check_attention(out, expect, bound)
    for b, n in enumerate(lengths):
        if n == 0:
            assert (out[b] == 0).all()
    again = decode_attention_q8(query.to(DEV), c, position.to(DEV), 1 / math.sqrt(dim))
    assert torch.equal(out, again)


def test_decode_attention_shared_position_and_long_rows():
    """One position for every row, more tiles than CTAs, so that units split over several."""
    from kernels.decode_attention import decode_attention_q8
    g = torch.Generator().manual_seed(3)
    cache = oq.random_cache(3, 2, 9000, 128, 64, g)
    position = torch.tensor([8990])
    poison(cache, position)
    query = torch.randn(3, 8, 1, 128, generator=g).bfloat16()
    expect, bound = oq.attention(query.transpose(1, 2), cache, position, 0.09)
    out = decode_attention_q8(query.to(DEV), handle(cache), position.to(DEV), 0.09)
    check_attention(out, expect, bound)


def test_decode_attention_ragged_batch_on_device():
    """64 ragged rows up to 5000 slots against a 32-bit product per row on the device. fp32 products
    sum up to 5000 terms: 2^-12 of the sizes at most, beside the bound's own terms."""
    from kernels.decode_attention import decode_attention_q8
    from kernels.quant import QuantCache
    g = torch.Generator(device=DEV).manual_seed(5)
    batch, kv_heads, groups, dim, capacity = 64, 8, 4, 128, 5000
    lengths = torch.randint(0, capacity + 1, (batch,), generator=torch.Generator().manual_seed(1))
    lengths[7] = 0
    codes = [(torch.randn(batch, kv_heads, capacity, dim, device=DEV, generator=g) * 100).clamp(-448, 448).to(oq.E4M3)
             for _ in range(2)]
    scales = [torch.exp2(torch.randint(-9, -5, (batch, kv_heads, -(-capacity // 64)), device=DEV, generator=g).float())
              for _ in range(2)]
    cache = QuantCache(*codes, *scales, 64)
    query = torch.randn(batch, kv_heads * groups, 1, dim, device=DEV, generator=g).bfloat16()
    out = decode_attention_q8(query, cache, (lengths - 1).to(DEV), 0.08).float()
    keys, values = cache.dequantized()
    for b, n in enumerate(lengths.tolist()):
        if n == 0:
            assert (out[b] == 0).all()
            continue
        q = query[b, :, 0].double().view(kv_heads, groups, dim)
        p = torch.softmax(torch.einsum("hgd,hnd->hgn", q, keys[b, :, :n].double()) * 0.08, -1)
        expect = torch.einsum("hgn,hnd->hgd", p, values[b, :, :n].double()).reshape(-1, dim)
        size = torch.einsum("hgn,hnd->hgd", p, values[b, :, :n].double().abs()).reshape(-1, dim)
        # P's f16 rounding: 2^-11, and 2^-25 of the row's largest p vs, at most 16 / n times their mean here
        tolerance = 2 ** -8 * expect.abs() + (2 ** -10 + 2 ** -12) * size
        assert ((out[b, 0].double() - expect).abs() <= tolerance).all(), b


def test_decode_attention_uneven_scales():
    """Blocks whose scales lie 2^40 apart, blocks of zeros (scale 2^-100 or 0), scales that are no
    powers of two: the value product's own pivot keeps each row's result."""
    from kernels.decode_attention import decode_attention_q8
    g = torch.Generator().manual_seed(8)
    cache = oq.random_cache(4, 2, 320, 64, 32, g)
    cache["value_scales"][0] = torch.exp2(torch.linspace(-30, 10, 10).round())
    cache["value_scales"][1, :, ::2] = 0.0
    cache["values"][2] = torch.zeros(2, 320, 64).to(oq.E4M3)
    cache["value_scales"][2] = 2.0 ** -100
    cache["value_scales"][3] *= 1.37
    cache["key_scales"][3] *= 0.81
    cache["key_scales"][1, :, 3] = 0.0
    position = torch.tensor([319, 300, 319, 257])
    query = (4 * torch.randn(4, 6, 1, 64, generator=g)).bfloat16()
    expect, bound = oq.attention(query.transpose(1, 2), cache, position, 0.125)
    out = decode_attention_q8(query.to(DEV), handle(cache), position.to(DEV), 0.125)
    check_attention(out, expect, bound + 1e-40)


@pytest.mark.parametrize("factor", [2.0 ** -90, 2.0 ** 60])
def test_decode_attention_query_range(factor):
    """Queries far outside f16's range (with a scale that undoes it)."""
    from kernels.decode_attention import decode_attention_q8
    g = torch.Generator().manual_seed(9)
    cache = oq.random_cache(2, 2, 200, 128, 16, g)
    position = torch.tensor([199, 60])
    query = torch.randn(2, 8, 1, 128, generator=g).bfloat16() * factor
    query[0, 0] = 0.0
    scale = 0.0883 / factor
    expect, bound = oq.attention(query.transpose(1, 2), cache, position, scale)
    check_attention(decode_attention_q8(query.to(DEV), handle(cache), position.to(DEV), scale), expect, bound)


@pytest.mark.parametrize("tokens,dim,batch", [(1, 128, 2), (1, 64, 40), (3, 128, 2), (5, 64, 40), (8, 128, 40)])
@pytest.mark.parametrize("factor", [2.0 ** 20, 2.0 ** 60])
def test_scores_whose_rounding_passes_one(tokens, dim, batch, factor):
    """Scores of 2^24 and more: the softmax is one slot, whose value comes back (each bf16 once rounded). Value
    scales far from 1 and in every block another must not turn the scores' rounding into a factor."""
    from kernels.decode_attention import block_attention_q8
    g = torch.Generator().manual_seed(tokens + batch)
    capacity, kv_heads, groups = 300, 4, 4
    cache = oq.random_cache(batch, kv_heads, capacity, dim, 16, g)
    blocks = cache["value_scales"].shape[2]
    cache["value_scales"] *= torch.exp2(torch.randint(-40, 40, (batch, kv_heads, blocks), generator=g).float())
    position = torch.randint(130, capacity - tokens, (batch,), generator=g)
    chain = torch.full((batch,), tokens)
    query = (torch.randn(batch, tokens, kv_heads * groups, dim, generator=g) * factor).bfloat16()
    out = block_attention_q8(query.to(DEV), handle(cache), position.to(DEV), 1.0, chain.to(DEV)).cpu().double()
    keys, values = (cache[name + "s"].double() * cache[name + "_scales"].double().repeat_interleave(
        16, 2)[:, :, :capacity, None] for name in ("key", "value"))
    checked = 0
    for b in range(batch):
        for t in range(tokens):
            n = int(position[b]) + t + 1
            q = query[b, t].double().view(kv_heads, groups, dim)
            scores = torch.einsum("hgd,hnd->hgn", q, keys[b, :, :n])
            best = scores.topk(2, -1)
            # fp32 sums of at most 128 exact products, then two roundings: 2^-15 of the two scores' sizes
            size = torch.einsum("hgd,hnd->hgn", q.abs(), keys[b, :, :n].abs()).amax(-1)
            clear = best.values[..., 0] - best.values[..., 1] > 2.0 ** -15 * size + 200
            expect = torch.gather(values[b, :, :n], 1, best.indices[..., :1].expand(-1, -1, dim))
            got = out[b, t].view(kv_heads, groups, dim)
            # P and the output round once each
            assert ((got - expect).abs() <= (2.0 ** -8 + 2.0 ** -10) * expect.abs())[clear].all(), (b, t)
            checked += int(clear.sum())
    assert checked > batch * tokens * kv_heads * groups // 2
    assert torch.isfinite(out).all()


def test_decode_attention_passes_nan_on():
    """A NaN in a slot that a row sees reaches that row's outputs, and no other row's."""
    from kernels.decode_attention import decode_attention_q8
    g = torch.Generator().manual_seed(10)
    cache = oq.random_cache(3, 1, 100, 64, 16, g)
    cache["keys"].view(torch.uint8)[0, 0, 40, 3] = 0x7f
    cache["values"].view(torch.uint8)[1, 0, 40, 3] = 0xff
    query = torch.randn(3, 2, 1, 64, generator=g).bfloat16()
    out = decode_attention_q8(query.to(DEV), handle(cache), torch.tensor([99, 99, 99]).to(DEV), 0.125).cpu()
    assert torch.isnan(out[0]).all()
    assert torch.isnan(out[1, ..., 3]).all() and torch.isfinite(out[1, ..., :3]).all()
    assert torch.isfinite(out[2]).all()


@pytest.mark.parametrize("batch,tokens,q_heads,kv_heads,dim,capacity,block,first,chain", [
    (8, 5, 32, 8, 128, 400, 64, [395, 0, 100, 127, 128, 200, 63, -1], [5, 3, 1, 2, 5, 4, 5, 5]),
    (2, 16, 16, 2, 64, 777, 32, [761, 300], [16, 7]),
    (2, 16, 16, 2, 128, 300, 16, [200, 120], [3, 16]),
    (3, 1, 8, 2, 128, 70, 64, [0, 63, 69], [1, 1, 1]),
    (2, 7, 7, 7, 64, 60, 16, [53, 11], [7, 2]),
    (1, 40, 4, 4, 128, 200, 64, [150], [11]),   # tokens past the 32nd column: several member groups
])
def test_block_attention(batch, tokens, q_heads, kv_heads, dim, capacity, block, first, chain):
    from kernels.decode_attention import block_attention_q8
    g = torch.Generator().manual_seed(tokens * capacity)
    cache = oq.random_cache(batch, kv_heads, capacity, dim, block, g)
    position, chain = torch.tensor(first), torch.tensor(chain)
    poison(cache, position, tokens)
    query = torch.randn(batch, tokens, q_heads, dim, generator=g).bfloat16()
    expect, bound = oq.attention(query, cache, position, 1 / math.sqrt(dim), chain)
    c = handle(cache)
    out = block_attention_q8(query.to(DEV), c, position.to(DEV), 1 / math.sqrt(dim), chain.to(DEV))
    assert out.shape == query.shape
    check_attention(out, expect, bound)
    assert torch.equal(out, block_attention_q8(query.to(DEV), c, position.to(DEV), 1 / math.sqrt(dim), chain.to(DEV)))


@pytest.mark.parametrize("dim", [64, 128])
def test_block_attention_hides_nan_of_later_drafts(dim):
    """A NaN key or value in a draft's slot stays with the tokens that see that slot."""
    from kernels.decode_attention import block_attention_q8
    g = torch.Generator().manual_seed(12)
    tokens, capacity = 6, 80
    cache = oq.random_cache(2, 2, capacity, dim, 16, g)
    position, chain = torch.tensor([62, 30]), torch.tensor([4, 6])
    poison(cache, position, tokens)
    sound = {k: v.clone() if torch.is_tensor(v) else v for k, v in cache.items()}
    cache["values"].view(torch.uint8)[0, :, 62 + 2, 5] = 0x7f   # draft 2: seen by tokens 2 and 3
    cache["keys"].view(torch.uint8)[1, :, 30 + 4, 1] = 0x7f     # draft 4: seen by tokens 4 and 5
    query = torch.randn(2, tokens, 8, dim, generator=g).bfloat16()
    expect, bound = oq.attention(query, sound, position, 0.1, chain)
    out = block_attention_q8(query.to(DEV), handle(cache), position.to(DEV), 0.1, chain.to(DEV)).cpu()
    assert torch.isnan(out[0, 2:4, :, 5]).all() and torch.isnan(out[1, 4:]).all()
    hidden = torch.ones_like(out, dtype=torch.bool)
    hidden[0, 2:4, :, 5] = False
    hidden[1, 4:] = False
    assert torch.isfinite(out[hidden]).all()
    assert ((out.double() - expect).abs()[hidden] <= bound[hidden]).all()


@pytest.mark.parametrize("tokens,dim", [(3, 64), (3, 128), (5, 64), (5, 128), (8, 64), (8, 128), (1, 128)])
def test_block_attention_many_ragged_rows(tokens, dim):
    """More units than SMs (slices of a persistent grid that split units and cross them), two to four column
    groups, rows from empty to several tiles."""
    from kernels.decode_attention import block_attention_q8
    g = torch.Generator().manual_seed(100 * tokens + dim)
    batch, capacity = 20, 700
    position = torch.randint(-1, capacity - tokens + 1, (batch,), generator=g)
    position[:4] = torch.tensor([-1, 0, capacity - tokens, 127])
    chain = torch.randint(1, tokens + 1, (batch,), generator=g)
    cache = oq.random_cache(batch, 8, capacity, dim, 32, g)
    poison(cache, position, tokens)
    query = torch.randn(batch, tokens, 32, dim, generator=g).bfloat16()
    expect, bound = oq.attention(query, cache, position, 1 / math.sqrt(dim), chain)
    out = block_attention_q8(query.to(DEV), handle(cache), position.to(DEV), 1 / math.sqrt(dim), chain.to(DEV))
    check_attention(out, expect, bound)
    assert (out[0] == 0).all()


@pytest.mark.parametrize("tokens,dim,q_heads", [(1, 64, 8), (2, 64, 48), (3, 128, 56), (4, 64, 64)])
def test_block_attention_slices_of_long_rows(tokens, dim, q_heads):
    """A capacity from which many units are cut into slices: a few long rows among short ones, one to four
    column groups, a NaN in one row's last draft."""
    from kernels.decode_attention import block_attention_q8
    g = torch.Generator().manual_seed(tokens * dim)
    batch, capacity, kv_heads = 19, 4800, 8
    position = torch.randint(-1, 400, (batch,), generator=g)
    position[3], position[4], position[11] = capacity - tokens, -1, 2000
    chain = torch.randint(1, tokens + 1, (batch,), generator=g)
    cache = oq.random_cache(batch, kv_heads, capacity, dim, 64, g)
    poison(cache, position, tokens)
    sound = {k: v.clone() if torch.is_tensor(v) else v for k, v in cache.items()}
    cache["values"].view(torch.uint8)[11, :, 2000 + tokens - 1, 9] = 0xff
    chain[11] = tokens
    query = torch.randn(batch, tokens, q_heads, dim, generator=g).bfloat16()
    expect, bound = oq.attention(query, sound, position, 1 / math.sqrt(dim), chain)
    out = block_attention_q8(query.to(DEV), handle(cache), position.to(DEV), 1 / math.sqrt(dim), chain.to(DEV)).cpu()
    assert torch.isnan(out[11, -1, :, 9]).all() and (out[4] == 0).all()
    kept = torch.ones_like(out, dtype=torch.bool)
    kept[11, -1, :, 9] = False
    assert torch.isfinite(out[kept]).all()
    assert ((out.double() - expect).abs()[kept] <= bound[kept]).all()


@pytest.mark.parametrize("batch", [2, 40])
@pytest.mark.parametrize("tokens,dim", [(1, 128), (3, 128), (5, 64), (7, 128)])
def test_block_attention_rising_scores_and_uneven_scales(batch, tokens, dim):
    """Scores that rise from block to block, so that the pivots move in every tile, and value scales 2^40
    apart, 2^-100 or 0, so that the value product's pivot moves on its own."""
    from kernels.decode_attention import block_attention_q8
    g = torch.Generator().manual_seed(batch + tokens)
    capacity, kv_heads = 800, 4
    cache = oq.random_cache(batch, kv_heads, capacity, dim, 64, g)
    blocks = cache["key_scales"].shape[2]
    cache["key_scales"] *= torch.exp2(torch.linspace(-2, 3, blocks).round())
    cache["value_scales"][0] = torch.exp2(torch.linspace(-30, 10, blocks).round())
    cache["value_scales"][1] = torch.exp2(torch.linspace(10, -30, blocks).round())
    cache["value_scales"][1, :, ::3] = 0.0
    if batch > 2:
        cache["value_scales"][2] = 0.0
        cache["values"][3] = torch.zeros(kv_heads, capacity, dim).to(oq.E4M3)
        cache["value_scales"][3] = 2.0 ** -100
        cache["value_scales"][4] *= 1.37
        cache["key_scales"][4] *= 0.81
    position = torch.full((batch,), capacity - tokens)
    chain = torch.full((batch,), tokens)
    query = torch.randn(batch, tokens, kv_heads * 4, dim, generator=g).bfloat16()
    expect, bound = oq.attention(query, cache, position, 1 / math.sqrt(dim), chain)
    out = block_attention_q8(query.to(DEV), handle(cache), position.to(DEV), 1 / math.sqrt(dim), chain.to(DEV))
    check_attention(out, expect, bound + 1e-40)


@pytest.mark.parametrize("tokens,dim", [(2, 128), (4, 64), (4, 128), (8, 128)])
def test_block_attention_hides_nan_in_many_rows(tokens, dim):
    """The same where slices of the grid end inside the rows, with the NaN in the last draft's slot."""
    from kernels.decode_attention import block_attention_q8
    g = torch.Generator().manual_seed(tokens + dim)
    batch, capacity = 24, 300
    position = torch.randint(0, capacity - tokens + 1, (batch,), generator=g)
    chain = torch.full((batch,), tokens)
    cache = oq.random_cache(batch, 8, capacity, dim, 16, g)
    poison(cache, position, tokens)
    sound = {k: v.clone() if torch.is_tensor(v) else v for k, v in cache.items()}
    for b in range(batch):
        cache["values"].view(torch.uint8)[b, :, int(position[b]) + tokens - 1, 9] = 0xff
    query = torch.randn(batch, tokens, 32, dim, generator=g).bfloat16()
    expect, bound = oq.attention(query, sound, position, 0.1, chain)
    out = block_attention_q8(query.to(DEV), handle(cache), position.to(DEV), 0.1, chain.to(DEV)).cpu()
    assert torch.isnan(out[:, -1, :, 9]).all()
    hidden = torch.ones_like(out, dtype=torch.bool)
    hidden[:, -1, :, 9] = False
    assert torch.isfinite(out[hidden]).all()
    assert ((out.double() - expect).abs()[hidden] <= bound[hidden]).all()


# ------------------------------------------------------------------------------ append
def append_case(batch, tokens, q_heads, kv_heads, dim, capacity, block, mode, starts, seed):
    g = torch.Generator().manual_seed(seed)
    packed = torch.randn(batch, tokens, (q_heads + 2 * kv_heads) * dim, generator=g).bfloat16()
    gains = [(1 + 0.2 * torch.randn(dim, generator=g)).bfloat16() for _ in range(2)]
    slots = torch.tensor(starts)[:, None] + torch.arange(tokens)  # [B, T] or [1, T]
    angle = slots[..., None].clamp_min(0).double() * 1e4 ** (-torch.arange(0, dim, 2).double() / dim)
    angle = torch.cat((angle, angle), -1)
    cos, sin = angle.cos().bfloat16(), angle.sin().bfloat16()
    cache = oq.random_cache(batch, kv_heads, capacity, dim, block, g)
    position = {"prefill": torch.arange(tokens), "decode": torch.tensor(starts[:1]), "rows": torch.tensor(starts)}[mode]
    return packed, gains, cos, sin, cache, position


def expected_append(packed, gains, cos, sin, cache, starts, q_heads, kv_heads, dim):
    batch, tokens, _ = packed.shape
    heads = packed.double().view(batch, tokens, q_heads + 2 * kv_heads, dim)
    cos, sin = cos.expand(batch, -1, -1)[:, :, None], sin.expand(batch, -1, -1)[:, :, None]
    query = oq.norm_rope(heads[:, :, :q_heads], gains[0], EPS, cos, sin)
    keys = oq.norm_rope(heads[:, :, q_heads:q_heads + kv_heads], gains[1], EPS, cos, sin)
    after = {k: v.clone() if torch.is_tensor(v) else v for k, v in cache.items()}
    real = {"key": oq.append(after, "key", keys, starts),
            "value": oq.append(after, "value", heads[:, :, q_heads + kv_heads:], starts)}
    return query, after, real


def check_append(cache, after, real, starts, tokens):
    """Scales, values and earlier or untouched codes to the bit. Keys pass fp32 arithmetic (noise below
    2^-18 of a head's largest value): within half an e4m3 step of the exact key, 2^-4 of it or
    2^-10 of the scale."""
    assert torch.equal(cache.key_scales.cpu(), after["key_scales"])
    assert torch.equal(cache.value_scales.cpu(), after["value_scales"])
    assert torch.equal(cache.values.cpu().view(torch.uint8), after["values"].view(torch.uint8))
    keys, block = cache.keys.cpu(), after["block"]
    capacity = keys.shape[2]
    written = torch.zeros(keys.shape[0], capacity, dtype=torch.bool)
    for b in range(keys.shape[0]):
        if starts[b] >= 0:
            written[b, starts[b]:starts[b] + tokens] = True
    hidden = ~written[:, None].expand(-1, keys.shape[1], -1)
    assert torch.equal(keys.view(torch.uint8)[hidden], after["keys"].view(torch.uint8)[hidden])
    per_slot = after["key_scales"].double().repeat_interleave(block, 2)[:, :, :capacity, None]
    value = keys.double() * per_slot
    exact = real["key"]
    noise = 2.0 ** -18 * exact.abs().amax(-1, keepdim=True)
    bound = torch.maximum(2.0 ** -4 * exact.abs(), 2.0 ** -10 * per_slot) + noise
    off = (value - exact).abs()[~hidden]
    assert (off <= bound[~hidden]).all()


@pytest.mark.parametrize("batch,tokens,q_heads,kv_heads,dim,capacity,block,mode,starts", [
    (3, 1, 8, 2, 128, 100, 64, "decode", [0]),
    (3, 1, 8, 2, 128, 100, 64, "decode", [63]),
    (3, 1, 8, 2, 128, 100, 64, "decode", [64]),
    (2, 1, 7, 1, 64, 33, 16, "decode", [32]),
    (2, 3, 4, 4, 128, 90, 32, "decode", [30]),          # three tokens that straddle a block
    (4, 1, 16, 8, 128, 200, 32, "rows", [0, 31, 199, -1]),
    (3, 40, 4, 2, 64, 300, 16, "rows", [7, 0, 250]),
    (2, 1, 4, 2, 128, 70, 64, "prefill", [0]),
    (2, 130, 6, 2, 128, 131, 64, "prefill", [0]),
    (1, 333, 4, 1, 64, 400, 32, "prefill", [0]),
])
def test_append(batch, tokens, q_heads, kv_heads, dim, capacity, block, mode, starts):
    from kernels.qk_rope import qk_rope_cache_q8
    packed, gains, cos, sin, cache, position = append_case(batch, tokens, q_heads, kv_heads, dim, capacity, block, mode,
                                                           starts, seed=capacity + tokens)
    full = starts if mode == "rows" else starts * batch
    query, after, real = expected_append(packed, gains, cos, sin, cache, full, q_heads, kv_heads, dim)
    c = handle(cache)
    norms = [SimpleNamespace(weight=w.to(DEV), variance_epsilon=EPS) for w in gains]
    out = qk_rope_cache_q8(packed.to(DEV), *norms, cos.to(DEV).contiguous(), sin.to(DEV).contiguous(), position.to(DEV),
                           c, q_heads, prefill=mode == "prefill", rows=mode == "rows")
    assert out.shape == (batch, q_heads, tokens, dim)
    out = out.transpose(1, 2).cpu().double()
    noise = 2.0 ** -18 * query.abs().amax(-1, keepdim=True)
    assert ((out - query).abs() <= 2.0 ** -8 * query.abs() + noise).all()
    check_append(c, after, real, full, tokens)


def test_append_one_token_at_a_time_matches_growing_rule():
    """20 tokens of growing size, one call each: codes and scales equal the rule applied step by step."""
    from kernels.qk_rope import qk_rope_cache_q8
    g = torch.Generator().manual_seed(4)
    batch, kv_heads, dim, block = 2, 2, 64, 16
    cache = oq.random_cache(batch, kv_heads, 40, dim, block, g)
    c = handle(cache)
    norms = [SimpleNamespace(weight=torch.ones(dim, dtype=torch.bfloat16, device=DEV), variance_epsilon=EPS)] * 2
    cos, sin = torch.ones(1, 1, dim, dtype=torch.bfloat16), torch.zeros(1, 1, dim, dtype=torch.bfloat16)
    for step in range(20):
        size = 2.0 ** (step % 9 - 3)
        packed = torch.randn(batch, 1, 6 * dim, generator=g).bfloat16()
        packed[..., 4 * dim:] *= size
        qk_rope_cache_q8(packed.to(DEV), *norms, cos.to(DEV), sin.to(DEV), torch.tensor([step + 3], device=DEV), c, 2)
        oq.append(cache, "value", packed.double().view(batch, 1, 6, dim)[:, :, 4:], [step + 3] * batch)
        assert torch.equal(c.value_scales.cpu(), cache["value_scales"]), step
        assert torch.equal(c.values.cpu().view(torch.uint8), cache["values"].view(torch.uint8)), step


def test_append_split_partials_tables_and_phases():
    """fp32 split partials sum, round to bf16 and continue as the bf16 input does; whole tables are
    read at the device-side position, and through a verify block's phases."""
    from kernels.merged import Split
    from kernels.qk_rope import qk_rope_cache_q8
    g = torch.Generator().manual_seed(6)
    batch, q_heads, kv_heads, dim, capacity = 3, 4, 2, 128, 96
    width = (q_heads + 2 * kv_heads) * dim
    partial = torch.randn(5, batch, width, generator=g).to(DEV)
    total = partial[0]
    for s in range(1, 5):
        total = total + partial[s]
    packed = total.bfloat16().view(batch, 1, width)
    norms = [SimpleNamespace(weight=(1 + 0.1 * torch.randn(dim, generator=g)).bfloat16().to(DEV), variance_epsilon=EPS)
             for _ in range(2)]
    cos, sin = (torch.randn(capacity, dim, generator=g).bfloat16().to(DEV) for _ in range(2))
    cache = oq.random_cache(batch, kv_heads, capacity, dim, 32, g)
    one, two, three = handle(cache), handle(cache), handle(cache)
    position = torch.tensor([41], device=DEV)
    a = qk_rope_cache_q8(packed, *norms, cos[41].view(1, 1, dim).contiguous(), sin[41].view(1, 1, dim).contiguous(),
                         position, one, q_heads)
    b = qk_rope_cache_q8(Split(partial, (batch, 1, width)), *norms, cos, sin, position, two, q_heads, table=True)
    rows = torch.tensor([40, 40, 40], device=DEV)
    c = qk_rope_cache_q8(packed, *norms, cos, sin, rows + 1, three, q_heads, rows=True,
                         phases=torch.zeros(batch, 1, dtype=torch.int64, device=DEV))
    for other, query in ((two, b), (three, c)):
        assert torch.equal(a, query)
        assert torch.equal(one.keys.view(torch.uint8), other.keys.view(torch.uint8))
        assert torch.equal(one.values.view(torch.uint8), other.values.view(torch.uint8))
        assert torch.equal(one.key_scales, other.key_scales) and torch.equal(one.value_scales, other.value_scales)


def test_append_not_finite_and_zero():
    """Infinities and NaN become the NaN code and set no scale; zeros get the least scale."""
    from kernels.qk_rope import qk_rope_cache_q8
    dim = 64
    cache = oq.empty_cache(1, 1, 20, dim, 16)
    c = handle(cache)
    packed = torch.ones(1, 1, 3 * dim).bfloat16()
    packed[..., 2 * dim] = float("inf")
    packed[..., 2 * dim + 1] = float("nan")
    packed[..., 2 * dim + 2] = -3.5
    norms = [SimpleNamespace(weight=torch.ones(dim, dtype=torch.bfloat16, device=DEV), variance_epsilon=EPS)] * 2
    cos, sin = torch.ones(1, 1, dim).bfloat16().to(DEV), torch.zeros(1, 1, dim).bfloat16().to(DEV)
    qk_rope_cache_q8(packed.to(DEV), *norms, cos, sin, torch.tensor([0], device=DEV), c, 1)
    assert float(c.value_scales[0, 0, 0]) == 2.0 ** -7  # 3.5 = 448 / 128
    values = c.dequantized()[1][0, 0, 0].cpu()
    assert torch.isnan(values[:2]).all() and float(values[2]) == -3.5 and (values[3:] == 1).all()
    packed[..., 2 * dim:] = 0
    qk_rope_cache_q8(packed.to(DEV), *norms, cos, sin, torch.tensor([16], device=DEV), c, 1)
    assert float(c.value_scales[0, 0, 1]) == 2.0 ** -100 and (c.dequantized()[1][0, 0, 16] == 0).all()


def test_append_past_the_cache_is_reported():
    from kernels import _native
    from kernels.qk_rope import qk_rope_cache_q8
    g = torch.Generator().manual_seed(2)
    cache = oq.random_cache(1, 1, 20, 64, 16, g)
    c = handle(cache)
    norms = [SimpleNamespace(weight=torch.ones(64, dtype=torch.bfloat16, device=DEV), variance_epsilon=EPS)] * 2
    cos = torch.ones(1, 1, 64).bfloat16().to(DEV)
    for start in (20, 31, 32, 10 ** 12):
        qk_rope_cache_q8(torch.randn(1, 1, 3 * 64, generator=g).bfloat16().to(DEV), *norms, cos, cos,
                         torch.tensor([start], device=DEV), c, 1)
        assert _native.device_error() != 0
        for name in ("keys", "values"):
            assert torch.equal(getattr(c, name).cpu().view(torch.uint8), cache[name].view(torch.uint8))


@pytest.mark.parametrize("dim,block", [(64, 16), (128, 64)])
def test_relocate(dim, block):
    from kernels.spec import relocate_q8
    g = torch.Generator().manual_seed(dim)
    planes, layers, batch, heads, capacity = 2, 3, 5, 2, 150
    parts = [oq.random_cache(batch, heads, capacity, dim, block, g) for _ in range(layers)]
    codes = torch.stack([torch.stack([p["keys"].view(torch.uint8) for p in parts]),
                         torch.stack([p["values"].view(torch.uint8) for p in parts])]).view(oq.E4M3)
    scales = torch.stack([torch.stack([p["key_scales"] for p in parts]), torch.stack([p["value_scales"] for p in parts])])
    move_from, move_to = torch.tensor([70, -1, 149, 128, 66]), torch.tensor([63, 5, 128, 127, 64])
    store, store_scales = codes.to(DEV), scales.to(DEV)
    oq.relocate(codes.view(planes * layers, batch, heads, capacity, dim),
                scales.view(planes * layers, batch, heads, -1), block, move_from, move_to)
    relocate_q8(store, store_scales, block, move_from.to(DEV), move_to.to(DEV))
    assert torch.equal(store_scales.cpu(), scales)
    assert torch.equal(store.cpu().view(torch.uint8), codes.view(torch.uint8))


# ------------------------------------------------------------------------------ 4-bit weights
def weights(n, k, group, seed):
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(-8, 8, (n, k), generator=g, dtype=torch.int8)
    scales = (0.002 + 0.01 * torch.rand(n, k // group, generator=g)).bfloat16()
    return codes, scales, g


@pytest.mark.parametrize("rows", [1, 2, 8, 9, 16, 17, 31, 33, 64])
@pytest.mark.parametrize("n,k,group", [(8, 32, 32), (24, 96, 32), (1000, 320, 64), (136, 1152, 128), (2048, 2048, 128),
                                       (72, 4128, 32)])
def test_linear(rows, n, k, group):
    from kernels.linear import linear
    from kernels.quant import pack_weight4
    codes, scales, g = weights(n, k, group, n + k)
    x = torch.randn(rows, k, generator=g).bfloat16()
    y, size = oq.linear(x, codes, scales)
    w = pack_weight4(codes.to(DEV), scales.to(DEV))
    out = linear(x.to(DEV), w)
    assert out.shape == (rows, n) and out.dtype == torch.bfloat16
    assert ((out.cpu().double() - y).abs() <= oq.linear_bound(y, size, k)).all()
    assert torch.equal(out, linear(x.to(DEV), w, split_ok=True))


def test_linear_zero_scales_range_and_nan():
    """Zero scales give zeros, scales and inputs at the ends of bf16's range stay exact, a NaN input
    stays in its row."""
    from kernels.linear import linear
    from kernels.quant import pack_weight4
    codes, scales, g = weights(64, 256, 64, 1)
    scales[:8] = 0
    scales[8:16] = 2.0 ** -120
    scales[16:24] = 2.0 ** 90
    x = torch.randn(5, 256, generator=g).bfloat16()
    x[1] *= 2.0 ** 20
    x[2] *= 2.0 ** -20
    y, size = oq.linear(x, codes, scales)
    w = pack_weight4(codes.to(DEV), scales.to(DEV))
    out = linear(x.to(DEV), w)
    assert ((out.cpu().double() - y).abs() <= oq.linear_bound(y, size, 256) + 2.0 ** -133).all()
    assert (out[:, :8] == 0).all()
    x[3, 100] = float("nan")
    bad = linear(x.to(DEV), w)
    assert torch.isnan(bad[3]).all()
    keep = [0, 1, 2, 4]
    assert torch.equal(bad[keep], out[keep])


def test_linear_forms():
    """fp32 and split outputs, SwiGLU on 64-row gate/up blocks, leading dimensions, many rows."""
    from kernels import linear as klinear
    from kernels.quant import pack_weight4
    codes, scales, g = weights(512, 640, 128, 2)
    w = pack_weight4(codes.to(DEV), scales.to(DEV))
    x = torch.randn(3, 4, 640, generator=g).bfloat16()
    y, size = oq.linear(x.view(12, 640), codes, scales)
    out = klinear.linear(x.to(DEV), w)
    assert out.shape == (3, 4, 512)
    flat = x.view(12, 640).to(DEV)
    for epilogue, shape in ((klinear.FP32_OUT, (12, 512)), (klinear.SPLITS_OUT, (1, 12, 512))):
        part = klinear.project(flat, w, epilogue)
        assert part.dtype == torch.float32 and part.shape == shape
        assert ((part.view(12, 512).cpu().double() - y).abs() <= oq.linear_bound(y, size, 640, rounded=False)).all()
        assert torch.equal(part.view(12, 512).bfloat16(), out.view(12, 512))
    gate_up = out.view(12, 4, 2, 64).float()
    gate, up = gate_up[:, :, 0], gate_up[:, :, 1]
    silu = (gate.double() / (1 + (-gate.double()).exp()))
    act = klinear.swiglu_linear(x.to(DEV), w).view(12, 4, 64).double()
    # silu and the product each round once to bf16; expf and the division are off by 2^-21 at most
    assert ((act - silu * up.double()).abs() <= (2.0 ** -8 * 2 + 2.0 ** -14) * (silu * up.double()).abs()).all()
    dense = codes.double() * scales.double().repeat_interleave(128, 1)
    assert torch.equal(w.dequantized().cpu(), dense.bfloat16())
    many = torch.randn(65, 640, generator=g).bfloat16()
    y, size = oq.linear(many, codes, scales)
    # the expanded weights round once to bf16: 2^-8 of each product
    off = (klinear.linear(many.to(DEV), w).cpu().double() - y).abs()
    assert (off <= oq.linear_bound(y, size, 640) + 2.0 ** -8 * size).all()
    assert klinear.linear(many[:0].to(DEV), w).shape == (0, 512)


def test_linear_strided_and_unaligned_input():
    from kernels.linear import linear
    from kernels.quant import pack_weight4
    codes, scales, g = weights(64, 128, 32, 3)
    w = pack_weight4(codes.to(DEV), scales.to(DEV))
    wide = torch.randn(6, 300, generator=g).bfloat16().to(DEV)
    expect = linear(wide[:, 5:133].contiguous(), w)
    assert torch.equal(linear(wide[:, 5:133], w), expect)
    flat = torch.empty(6 * 128 + 3, dtype=torch.bfloat16, device=DEV)
    flat[3:].view(6, 128).copy_(wide[:, 5:133])
    assert torch.equal(linear(flat[3:].view(6, 128), w), expect)


def test_quantize_weight4_is_nearest():
    from kernels.quant import quantize_weight4
    g = torch.Generator().manual_seed(7)
    weight = (0.02 * torch.randn(48, 256, generator=g)).bfloat16()
    weight[3, 64:128] = 0
    w = quantize_weight4(weight.to(DEV), 64).dequantized().cpu().double()
    parts = weight.double().view(48, 4, 64)
    step = (parts.abs().amax(-1) / 7).float().bfloat16().double()
    # half a step (the largest may pass 7 steps by the scale's own rounding, 2^-8 of 7 steps), and
    # the expansion's rounding
    off = (w.view(48, 4, 64) - parts).abs()
    assert (off <= (0.5 + 7 * 2.0 ** -8) * step[..., None] + 2.0 ** -8 * parts.abs() + 1e-12).all()
    assert (w.view(48, 4, 64)[3, 1] == 0).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_quantize_weight4_refuses_what_is_not_finite(bad):
    from kernels.quant import quantize_weight4
    weight = torch.ones(16, 128, dtype=torch.bfloat16, device=DEV)
    weight[9, 70] = bad
    with pytest.raises(ValueError):
        quantize_weight4(weight, 64)


@pytest.mark.parametrize("code", [-9, 8])
def test_pack_weight4_refuses_codes_out_of_range(code):
    from kernels.quant import pack_weight4
    codes = torch.zeros(8, 64, dtype=torch.int8, device=DEV)
    codes[7, 63] = code
    with pytest.raises(ValueError):
        pack_weight4(codes, torch.ones(8, 1, dtype=torch.bfloat16, device=DEV))


@pytest.mark.parametrize("rows", [65, 100, 128, 129, 300])
def test_linear_more_rows_than_a_launch_takes(rows):
    """Two launches up to 128 rows, expanded weights above (rounded once to bf16: 2^-8 of each product)."""
    from kernels import linear as klinear
    from kernels.quant import pack_weight4
    codes, scales, g = weights(256, 320, 64, rows)
    w = pack_weight4(codes.to(DEV), scales.to(DEV))
    x = torch.randn(rows, 320, generator=g).bfloat16()
    y, size = oq.linear(x, codes, scales)
    expanded = 0.0 if rows <= 128 else 2.0 ** -8
    assert ((klinear.linear(x.to(DEV), w).cpu().double() - y).abs() <= oq.linear_bound(y, size, 320) + expanded * size).all()
    if rows > 128:
        with pytest.raises(ValueError):
            klinear.swiglu_linear(x.to(DEV), w)
        return
    for epilogue in (klinear.BF16_OUT, klinear.FP32_OUT, klinear.SPLITS_OUT, klinear.SWIGLU_OUT):
        whole = klinear.project(x.to(DEV), w, epilogue)
        parts = [klinear.project(x[a:b].contiguous().to(DEV), w, epilogue) for a, b in ((0, 64), (64, rows))]
        assert torch.equal(whole, torch.cat(parts, 1 if epilogue == klinear.SPLITS_OUT else 0))


def test_calls_on_two_streams_at_once():
    """Calls that overlap on the GPU share nothing: the results are those of calls in turn."""
    from kernels.decode_attention import block_attention_q8, decode_attention_q8
    from kernels.linear import linear
    from kernels.quant import quantize_weight4
    g = torch.Generator().manual_seed(31)
    jobs = []
    for i in range(2):
        small, large = (handle(oq.random_cache(b, 8, 600, 128, 64, g)) for b in (2, 24))
        w = quantize_weight4(torch.randn(2048, 1024, generator=g).bfloat16().to(DEV), 64)
        x = torch.randn(7 + i, 1024, generator=g).bfloat16().to(DEV)
        q = torch.randn(24, 5, 32, 128, generator=g).bfloat16().to(DEV)
        first = torch.randint(0, 595, (24,), generator=g).to(DEV)
        chain = torch.full((24,), 5).to(DEV)

        def job(small=small, large=large, w=w, x=x, q=q, first=first, chain=chain):
            one = q[:, :1].transpose(1, 2).contiguous()
            return (linear(x, w), decode_attention_q8(one[:2], small, first[:2], 0.09),
                    block_attention_q8(q[:2].contiguous(), small, first[:2], 0.09, chain[:2]),
                    decode_attention_q8(one, large, first, 0.09), block_attention_q8(q, large, first, 0.09, chain))

        jobs.append(job)
    expect = [job() for job in jobs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in jobs], [[], []]
    for _ in range(10):
        for i, job in enumerate(jobs):
            with torch.cuda.stream(streams[i]):
                got[i].append(job())
    torch.cuda.synchronize()
    for want, runs in zip(expect, got):
        for run in runs:
            for a, b in zip(want, run):
                assert torch.equal(a, b)


def test_first_calls_of_a_shape_inside_a_capture():
    """Shapes that no eager call has met: captured, replayed on new inputs, equal to eager calls after it."""
    from kernels.decode_attention import block_attention_q8, decode_attention_q8
    from kernels.linear import linear
    from kernels.quant import quantize_weight4
    g = torch.Generator().manual_seed(41)
    cache = handle(oq.random_cache(37, 8, 5200, 64, 32, g))  # the persistent form: a workspace of the graph's pool
    w = quantize_weight4(torch.randn(264, 416, generator=g).bfloat16().to(DEV), 32)
    x = torch.randn(3, 416, generator=g).bfloat16().to(DEV)
    q = torch.randn(37, 2, 24, 64, generator=g).bfloat16().to(DEV)
    position = torch.randint(-1, 5198, (37,), generator=g).to(DEV)
    chain = torch.full((37,), 2).to(DEV)
    one = q[:, :1].transpose(1, 2).contiguous()

    def calls():
        return (linear(x, w), decode_attention_q8(one, cache, position, 0.125),
                block_attention_q8(q, cache, position, 0.125, chain))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        captured = calls()
    for seed in range(2):
        x.copy_(torch.randn(3, 416, generator=g).bfloat16())
        one.copy_(torch.randn(37, 24, 1, 64, generator=g).bfloat16())
        q.copy_(torch.randn(37, 2, 24, 64, generator=g).bfloat16())
        position.copy_(torch.randint(-1, 5198, (37,), generator=g))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, calls()):
            assert torch.equal(a, b)
