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


# ------------------------------------------------------------------ the grid of slices and its merge
def stretched(cache, position, tokens, capacity=LONG):
    """The cache at a larger capacity, NaN codes and scales in every slot behind each row's last token."""
    out = {"block": cache["block"]}
    block, short = cache["block"], cache["keys"].shape[2]
    for name in ("key", "value"):
        batch, heads, _, dim = cache[name + "s"].shape
        codes = torch.full((batch, heads, capacity, dim), 0x7f, dtype=torch.uint8)
        scales = torch.full((batch, heads, -(-capacity // block)), float("nan"))
        for b in range(batch):
            p = int(position[b if len(position) > 1 else 0])
            end = 0 if p < 0 else min(p + tokens, short)
            codes[b, :, :end] = cache[name + "s"].view(torch.uint8)[b, :, :end]
            scales[b, :, :-(-end // block)] = cache[name + "_scales"][b, :, :-(-end // block)]
        out[name + "s"], out[name + "_scales"] = codes.view(oq.E4M3), scales
    return out


def sliced_handle(cache, position, tokens, q_heads):
    c = handle(stretched(cache, position, tokens))
    assert c.workspace_bytes(tokens, q_heads) > 0  # the form these tests are about
    return c


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("tokens,q_heads", [(1, 32), (1, 72), (3, 32), (2, 80), (5, 40), (4, 64), (6, 48)])
def test_slices_of_ragged_rows(tokens, q_heads, dim):
    """One to four column groups (and two member groups), rows from empty to six tiles: slices end inside units
    and cross them."""
    from kernels.decode_attention import block_attention_q8
    g = torch.Generator().manual_seed(100 * tokens + dim + q_heads)
    batch, kv_heads, capacity = 20, 8, 700
    position = torch.randint(-1, capacity - tokens + 1, (batch,), generator=g)
    position[:4] = torch.tensor([-1, 0, capacity - tokens, 127])
    chain = torch.randint(1, tokens + 1, (batch,), generator=g)
    cache = oq.random_cache(batch, kv_heads, capacity, dim, 32, g)
    query = torch.randn(batch, tokens, q_heads, dim, generator=g).bfloat16()
    expect, bound = oq.attention(query, cache, position, 1 / math.sqrt(dim), chain)
    c = sliced_handle(cache, position, tokens, q_heads)
    out = block_attention_q8(query.to(DEV), c, position.to(DEV), 1 / math.sqrt(dim), chain.to(DEV))
    check(out, expect, bound)
    assert (out[0] == 0).all()
    again = block_attention_q8(query.to(DEV), c, position.to(DEV), 1 / math.sqrt(dim), chain.to(DEV))
    assert torch.equal(out, again)


@pytest.mark.parametrize("dim,q_heads", [(64, 16), (128, 96)])
@pytest.mark.parametrize("lengths", [{}, {3: 1}, {0: 128}, {19: 129, 7: 16}, {2: 300, 11: 1, 12: 40}])
def test_slices_fewer_than_ctas(lengths, dim, q_heads):
    """Fewer tiles than CTAs, down to none: most slices are empty, and every row without a slot gives zeros."""
    from kernels.decode_attention import decode_attention_q8
    g = torch.Generator().manual_seed(dim + len(lengths))
    batch, kv_heads = 20, 8
    position = torch.full((batch,), -1)
    for b, n in lengths.items():
        position[b] = n - 1
    cache = oq.random_cache(batch, kv_heads, 320, dim, 16, g)
    query = torch.randn(batch, q_heads, 1, dim, generator=g).bfloat16()
    expect, bound = oq.attention(query.transpose(1, 2), cache, position, 0.1)
    c = sliced_handle(cache, position, 1, q_heads)
    out = decode_attention_q8(query.to(DEV), c, position.to(DEV), 0.1)
    check(out, expect, bound)
    assert (out[position.to(DEV) < 0] == 0).all()


@pytest.mark.parametrize("position", [-1, 0, 128, 611])
def test_slices_at_a_shared_position(position):
    from kernels.decode_attention import decode_attention_q8
    g = torch.Generator().manual_seed(position + 2)
    batch, kv_heads, dim, position = 20, 8, 128, torch.tensor([position])
    cache = oq.random_cache(batch, kv_heads, 640, dim, 64, g)
    query = torch.randn(batch, 32, 1, dim, generator=g).bfloat16()
    expect, bound = oq.attention(query.transpose(1, 2), cache, position, 0.09)
    c = sliced_handle(cache, position, 1, 32)
    check(decode_attention_q8(query.to(DEV), c, position.to(DEV), 0.09), expect, bound)


@pytest.mark.parametrize("tokens,dim", [(1, 128), (1, 64), (3, 128), (4, 64), (5, 64), (7, 128)])
def test_slices_of_rising_scores_and_uneven_scales(tokens, dim):
    """Scores that rise from block to block, so that the pivots move in every tile and differ between the runs
    that are merged, and value scales 2^40 apart, 2^-100 or 0, so that the value product's pivot moves on its
    own."""
    from kernels.decode_attention import block_attention_q8
    g = torch.Generator().manual_seed(dim + tokens)
    batch, capacity, kv_heads = 40, 800, 4
    cache = oq.random_cache(batch, kv_heads, capacity, dim, 64, g)
    blocks = cache["key_scales"].shape[2]
    cache["key_scales"] *= torch.exp2(torch.linspace(-2, 3, blocks).round())
    cache["value_scales"][0] = torch.exp2(torch.linspace(-30, 10, blocks).round())
    cache["value_scales"][1] = torch.exp2(torch.linspace(10, -30, blocks).round())
    cache["value_scales"][1, :, ::3] = 0.0
    cache["value_scales"][2] = 0.0
    cache["values"][3] = torch.zeros(kv_heads, capacity, dim).to(oq.E4M3)
    cache["value_scales"][3] = 2.0 ** -100
    cache["value_scales"][4] *= 1.37
    cache["key_scales"][4] *= 0.81
    position = torch.full((batch,), capacity - tokens)
    position[5:] = torch.randint(400, capacity - tokens + 1, (batch - 5,), generator=g)
    chain = torch.full((batch,), tokens)
    query = torch.randn(batch, tokens, kv_heads * 4, dim, generator=g).bfloat16()
    expect, bound = oq.attention(query, cache, position, 1 / math.sqrt(dim), chain)
    c = sliced_handle(cache, position, tokens, kv_heads * 4)
    out = block_attention_q8(query.to(DEV), c, position.to(DEV), 1 / math.sqrt(dim), chain.to(DEV))
    check(out, expect, bound + 1e-40)


@pytest.mark.parametrize("tokens,dim", [(2, 128), (4, 64), (4, 128), (8, 128)])
def test_slices_hide_nan_of_the_last_draft(tokens, dim):
    """A NaN in the last draft's slot stays with the token that sees it, where slices end inside the rows."""
    from kernels.decode_attention import block_attention_q8
    g = torch.Generator().manual_seed(tokens + dim)
    batch, capacity = 24, 300
    position = torch.randint(0, capacity - tokens + 1, (batch,), generator=g)
    chain = torch.full((batch,), tokens)
    sound = oq.random_cache(batch, 8, capacity, dim, 16, g)
    cache = {k: v.clone() if torch.is_tensor(v) else v for k, v in sound.items()}
    for b in range(batch):
        cache["values"].view(torch.uint8)[b, :, int(position[b]) + tokens - 1, 9] = 0xff
    query = torch.randn(batch, tokens, 32, dim, generator=g).bfloat16()
    expect, bound = oq.attention(query, sound, position, 0.1, chain)
    c = sliced_handle(cache, position, tokens, 32)
    out = block_attention_q8(query.to(DEV), c, position.to(DEV), 0.1, chain.to(DEV)).cpu()
    assert torch.isnan(out[:, -1, :, 9]).all()
    hidden = torch.ones_like(out, dtype=torch.bool)
    hidden[:, -1, :, 9] = False
    assert torch.isfinite(out[hidden]).all()
    assert ((out.double() - expect).abs()[hidden] <= bound[hidden]).all()


def sliced_jobs(g):
    """Two calls' inputs over caches whose attention takes partials."""
    from kernels.decode_attention import block_attention_q8, decode_attention_q8
    jobs = []
    for _ in range(2):
        position = torch.randint(0, 595, (24,), generator=g)
        c = sliced_handle(oq.random_cache(24, 8, 600, 128, 64, g), position, 5, 32)
        assert c.workspace_bytes(1, 32) > 0
        q = torch.randn(24, 5, 32, 128, generator=g).bfloat16().to(DEV)
        one, chain, at = q[:, :1].transpose(1, 2).contiguous(), torch.full((24,), 5).to(DEV), position.to(DEV)
        jobs.append(lambda c=c, q=q, one=one, chain=chain, at=at: (decode_attention_q8(one, c, at, 0.09),
                                                                   block_attention_q8(q, c, at, 0.09, chain)))
    return jobs


def test_slices_on_two_streams_at_once():
    """Calls that overlap on the GPU share no partials: the results are those of calls in turn."""
    jobs = sliced_jobs(torch.Generator().manual_seed(31))
    expect = [job() for job in jobs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in jobs], [[], []]
    for _ in range(20):
        for i, job in enumerate(jobs):
            with torch.cuda.stream(streams[i]):
                got[i].append(job())
    torch.cuda.synchronize()
    for want, runs in zip(expect, got):
        for run in runs:
            assert all(torch.equal(a, b) for a, b in zip(want, run))


def test_slices_of_two_graphs_and_eager_calls():
    """Two graphs on one cache handle, replayed on two streams at once beside eager calls on it."""
    job, other = sliced_jobs(torch.Generator().manual_seed(32))
    expect, beside = job(), other()
    torch.cuda.synchronize()
    streams, graphs, outs = [torch.cuda.Stream() for _ in range(2)], [], []
    for stream in streams:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            outs.append(job())
        graphs.append(graph)
    eager = []
    for _ in range(20):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        eager.append((job(), other()))
    torch.cuda.synchronize()
    for got, want in (*((o, expect) for o in outs), *((e, expect) for e, _ in eager), *((e, beside) for _, e in eager)):
        assert all(torch.equal(a, b) for a, b in zip(got, want))


# ------------------------------------------------------------------------------ append
@pytest.mark.parametrize("tokens", [1, 40])
@pytest.mark.parametrize("start", [70, 79, 80, 2 ** 61, 2 ** 62, 2 ** 63 - 70, 2 ** 63 - 2, 2 ** 63 - 1])
def test_append_past_the_cache_writes_nothing(start, tokens):
    """From the first slot past the cache (in its last block, whose scale is 0 here) to positions whose sum with
    the token count leaves 64 bits: neither codes nor scales change, the error word is set, and the queries are
    those of the same phases."""
    from types import SimpleNamespace
    from kernels import _native
    from kernels.qk_rope import qk_rope_cache_q8
    g = torch.Generator().manual_seed(tokens)
    cache = oq.random_cache(1, 1, 70, 64, 16, g)
    cache["key_scales"][..., -1] = cache["value_scales"][..., -1] = 0
    c = handle(cache)
    norms = [SimpleNamespace(weight=torch.ones(64, dtype=torch.bfloat16, device=DEV), variance_epsilon=1e-6)] * 2
    packed = torch.randn(1, tokens, 3 * 64, generator=g).bfloat16().to(DEV)
    cos, sin = (torch.randn(1, tokens, 64, generator=g).bfloat16().to(DEV) for _ in range(2))
    out = qk_rope_cache_q8(packed, *norms, cos, sin, torch.tensor([start], device=DEV), c, 1)
    assert _native.device_error() != 0
    for name in ("keys", "values"):
        assert torch.equal(getattr(c, name).cpu().view(torch.uint8), cache[name].view(torch.uint8))
        assert torch.equal(getattr(c, name[:-1] + "_scales").cpu(), cache[name[:-1] + "_scales"])
    assert torch.equal(out, qk_rope_cache_q8(packed, *norms, cos, sin, torch.tensor([0], device=DEV), c, 1))


@pytest.mark.parametrize("phase", [-2 ** 63, -43, 30, 2 ** 63 - 1])
def test_append_clamps_phases_outside_the_tables(phase):
    """A phase that leaves the tables is reported and read at the nearest end, whatever it adds up to."""
    from types import SimpleNamespace
    from kernels import _native
    from kernels.qk_rope import qk_rope_cache_q8
    g = torch.Generator().manual_seed(3)
    one, two = (oq.random_cache(2, 1, 70, 64, 16, torch.Generator().manual_seed(5)) for _ in range(2))
    a, b = handle(one), handle(two)
    norms = [SimpleNamespace(weight=torch.ones(64, dtype=torch.bfloat16, device=DEV), variance_epsilon=1e-6)] * 2
    packed = torch.randn(2, 1, 4 * 64, generator=g).bfloat16().to(DEV)
    cos, sin = (torch.randn(70, 64, generator=g).bfloat16().to(DEV) for _ in range(2))
    at = torch.tensor([41, 42], device=DEV)
    nearest = torch.full((2, 1), 0 if phase < 0 else 69, device=DEV)
    query = qk_rope_cache_q8(packed, *norms, cos, sin, at, a, 2, rows=True, phases=torch.full((2, 1), phase, device=DEV))
    assert _native.device_error() != 0
    expect = qk_rope_cache_q8(packed, *norms, cos, sin, at, b, 2, rows=True, phases=nearest - at[:, None])
    assert torch.equal(query, expect)
    for name in ("keys", "values"):
        assert torch.equal(getattr(a, name).view(torch.uint8), getattr(b, name).view(torch.uint8))


@pytest.mark.parametrize("sliced", [False, True])
def test_chains_longer_than_the_block(sliced):
    """A chain of any length from the block's on is the whole block."""
    from kernels.decode_attention import block_attention_q8
    g = torch.Generator().manual_seed(17)
    batch, kv_heads, tokens = (20, 8, 4) if sliced else (3, 2, 4)
    position = torch.randint(0, 290, (batch,), generator=g)
    cache = oq.random_cache(batch, kv_heads, 300, 64, 32, g)
    query = torch.randn(batch, tokens, kv_heads * 2, 64, generator=g).bfloat16()
    whole = torch.full((batch,), tokens)
    expect, bound = oq.attention(query, cache, position, 0.125, whole)
    c = sliced_handle(cache, position, tokens, kv_heads * 2) if sliced else handle(cache)
    for length in (tokens, 7, 2 ** 31, 2 ** 32, 2 ** 32 + 1, 2 ** 63 - 1):
        out = block_attention_q8(query.to(DEV), c, position.to(DEV), 0.125, torch.full((batch,), length).to(DEV))
        check(out, expect, bound)


# ------------------------------------------------------------------------------ 4-bit weights
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_pack_weight4_refuses_scales_that_are_not_finite(bad):
    from kernels.quant import pack_weight4
    codes = torch.zeros(16, 128, dtype=torch.int8, device=DEV)
    scales = torch.ones(16, 2, dtype=torch.bfloat16, device=DEV)
    pack_weight4(codes, scales)
    scales[11, 1] = bad
    with pytest.raises(ValueError):
        pack_weight4(codes, scales)


# ------------------------------------------------------------------------------ far slots
@pytest.mark.parametrize("tokens", [1, 3])
def test_offsets_past_32_bits(tokens):
    """Codes past 2^32 bytes into the cache: an append at the last slots, attention over rows of 1.9 and 2.2
    million slots whose keys are zero but for the appended ones and whose values are 1 / 128, and moves there and
    back. Tolerance: the output's rounding, and of the sizes 2^-11 for P, 2^-11.5 for scores up to 45 summed over 128
    dims in fp32, 2^-11.9 for 2200 fp32 sums a warp: below 2^-9 together."""
    from types import SimpleNamespace
    from kernels.decode_attention import block_attention_q8
    from kernels.qk_rope import qk_rope_cache_q8
    from kernels.quant import QuantCache
    from kernels.spec import relocate_q8
    batch, kv_heads, groups, dim, capacity, block = 2, 8, 2, 128, 2_200_003, 64
    g = torch.Generator(device=DEV).manual_seed(6)
    store = torch.zeros(2, 1, batch, kv_heads, capacity, dim, dtype=torch.uint8, device=DEV)
    store[1].fill_(0x38)  # the code of 1
    store = store.view(oq.E4M3)
    scales = torch.full((2, 1, batch, kv_heads, -(-capacity // block)), 2.0 ** -7, device=DEV)
    c = QuantCache(store[0, 0], store[1, 0], scales[0, 0], scales[1, 0], block)
    assert c.keys.numel() > 2 ** 32
    starts = [capacity - tokens, 1_900_001]
    position = torch.tensor(starts, device=DEV)
    packed = torch.randn(batch, tokens, (groups + 2) * kv_heads * dim, device=DEV, generator=g).bfloat16()
    norm = SimpleNamespace(weight=torch.ones(dim, dtype=torch.bfloat16, device=DEV), variance_epsilon=1e-6)
    cos, sin = (torch.full((batch, tokens, dim), v, device=DEV).bfloat16() for v in (1.0, 0.0))
    query = qk_rope_cache_q8(packed, norm, norm, cos, sin, position, c, groups * kv_heads, rows=True).transpose(1, 2)
    new = packed.view(batch, tokens, (groups + 2) * kv_heads, dim)[:, :, (groups + 1) * kv_heads:]
    out = block_attention_q8(query, c, position, 1.0, torch.full((batch,), tokens, device=DEV))

    def held(codes, scale, b, low, high):  # [Hkv, slots, D]: what slots of one block or two stand for
        at = torch.arange(low, high, device=DEV)
        return codes[b, :, low:high].double() * scale[b][:, at // block, None].double()

    for b, low in enumerate(starts):
        keys, values = (held(*x, b, low, low + tokens) for x in ((c.keys, c.key_scales), (c.values, c.value_scales)))
        want = new[b].transpose(0, 1).double()
        step = c.value_scales[b][:, torch.arange(low, low + tokens, device=DEV) // block, None].double()
        assert ((values - want).abs() <= torch.maximum(2.0 ** -4 * want.abs(), 2.0 ** -10 * step)).all()
        assert (held(c.values, c.value_scales, b, low - 2, low) == 2.0 ** -7).all()
        for t in range(tokens):
            q = query[b, t].double().view(kv_heads, groups, dim)
            p = torch.exp(torch.einsum("hgd,htd->hgt", q, keys[:, :t + 1]))
            total = low + p.sum(-1, keepdim=True)
            expect = (low * 2.0 ** -7 + torch.einsum("hgt,htd->hgd", p, values[:, :t + 1])) / total
            size = (low * 2.0 ** -7 + torch.einsum("hgt,htd->hgd", p, values[:, :t + 1].abs())) / total
            off = (out[b, t].double().view(kv_heads, groups, dim) - expect).abs()
            assert (off <= 2.0 ** -8 * expect.abs() + 2.0 ** -9 * size).all(), (b, t)
    c.values.view(torch.uint8)[1, :, capacity - 9] = 0x40  # 2
    relocate_q8(store, scales, block, torch.tensor([40, capacity - 9], device=DEV),
                torch.tensor([capacity - 1, 40], device=DEV))
    assert (held(c.values, c.value_scales, 0, capacity - 1, capacity) == 2.0 ** -7).all()
    assert (held(c.values, c.value_scales, 1, 40, 41) == 2.0 ** -6).all()
    del store, c
    torch.cuda.empty_cache()
