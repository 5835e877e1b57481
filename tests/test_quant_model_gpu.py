"""The quantised operators together, as the decode step runs them: DecodeState with an 8-bit cache, 4-bit
weights and both, eager, captured and composed by hand from the public calls."""

import math
from types import SimpleNamespace

import pytest
import torch

import cases
import decode as fdecode
import qwen3
from oracle import quant as oq

pytestmark = pytest.mark.gpu
DEV = "cuda"
FORMS = [("q8", 0), ("bf16", 64), ("q8", 32)]


@pytest.fixture(autouse=True)
def _no_device_errors():
    from kernels import _native
    _native.device_error()
    yield
    assert _native.device_error() == 0, "a kernel raised its device error word"


def tiny(group):
    cfg = qwen3.Config.make(**cases.TINY_QWEN3)
    weights = qwen3.from_state_dict(cfg, cases.tiny_qwen3_weights(), DEV)
    return qwen3.quantize_weights(weights, group) if group else weights


def state_of(weights, prompt, steps, kv_cache):
    return fdecode.DecodeState(weights, prompt.shape[0], prompt.shape[1], steps + 4, kv_cache=kv_cache, kv_block=16)


@pytest.mark.parametrize("kv_cache,group", FORMS)
def test_decode_state_graph_matches_eager(kv_cache, group):
    prompt, steps = cases.model_prompt(cases.MODEL_CASES[1])
    weights = tiny(group)
    eager = state_of(weights, prompt, steps, kv_cache)
    tokens, logits = fdecode.greedy(eager, prompt.to(DEV), steps)
    assert torch.isfinite(logits).all()
    state = state_of(weights, prompt, steps, kv_cache)
    state.prefill(prompt.to(DEV))
    seen = [state.token_ids[:, 0].clone()]
    state.capture()
    for _ in range(steps - 1):
        state.step()
        seen.append(state.token_ids[:, 0].clone())
    torch.cuda.synchronize()
    assert torch.equal(torch.stack(seen, 1), tokens)
    state.release()
    # a second generation on the same state starts its blocks anew
    again, logits2 = fdecode.greedy(eager, prompt.to(DEV), steps)
    assert torch.equal(again, tokens) and torch.equal(logits2, logits)


def test_decode_state_step_is_its_public_calls():
    """One step with both forms equals the same calls made by hand, bit for bit."""
    from kernels.decode_attention import decode_attention_q8
    from kernels.linear import linear, swiglu_linear
    from kernels.qk_rope import qk_rope_cache_q8
    from kernels.rmsnorm import add_rms_norm, embed_rms_norm
    prompt, steps = cases.model_prompt(cases.MODEL_CASES[1])
    weights = tiny(32)
    state, hand = (state_of(weights, prompt, steps, "q8") for _ in range(2))
    for s in (state, hand):
        s.prefill(prompt.to(DEV))
    state.decode(keep_logits=True)
    cfg, eps = weights.cfg, weights.cfg.rms_norm_eps
    x, residual = embed_rms_norm(hand.token_ids, weights.embed, weights.layers[0].ln1, eps)
    for i, layer in enumerate(weights.layers):
        cache = hand.cache.layers[i]
        norms = [SimpleNamespace(weight=w, variance_epsilon=eps) for w in (layer.q_norm, layer.k_norm)]
        query = qk_rope_cache_q8(linear(x, layer.qkv), *norms, hand.cos, hand.sin, hand.position, cache, weights.q_heads,
                                 table=True)
        a = decode_attention_q8(query, cache, hand.position, 1 / math.sqrt(cfg.head_dim))
        x, residual = add_rms_norm(linear(a.reshape(hand.batch, 1, -1), layer.o), residual, layer.ln2, eps)
        following = weights.layers[i + 1].ln1 if i + 1 < len(weights.layers) else weights.final_norm
        x, residual = add_rms_norm(linear(swiglu_linear(x, layer.gate_up), layer.down), residual, following, eps)
        assert torch.equal(cache.keys.view(torch.uint8), state.cache.layers[i].keys.view(torch.uint8))
        assert torch.equal(cache.value_scales, state.cache.layers[i].value_scales)
    logits = linear(x, weights.lm_head)
    # the LM head's split count differs between the two calls: fp32 sums in another order, one rounding each
    scale = logits.float().abs().max()
    assert ((logits.float() - state.logits.float()).abs() <= 2 ** -7 * scale).all()


def test_chain_of_stages_within_bounds():
    """qkv projection (4-bit) -> append -> attention -> o projection (4-bit): each stage against its 64-bit
    restatement on the stage's own inputs, ragged rows, an inactive one, a block that is joined."""
    from kernels.decode_attention import decode_attention_q8
    from kernels.linear import linear
    from kernels.qk_rope import qk_rope_cache_q8
    from kernels.quant import QuantCache, pack_weight4
    g = torch.Generator().manual_seed(21)
    batch, hq, hkv, dim, capacity, block, hidden = 5, 8, 2, 64, 150, 32, 256
    position = torch.tensor([149, 0, 31, 32, -1])

    def weight(n, k):
        codes = torch.randint(-8, 8, (n, k), generator=g, dtype=torch.int8)
        return codes, (0.01 + 0.01 * torch.rand(n, k // 64, generator=g)).bfloat16()

    wqkv, wo = weight((hq + 2 * hkv) * dim, hidden), weight(hidden, hq * dim)
    pq, po = (pack_weight4(c.to(DEV), s.to(DEV)) for c, s in (wqkv, wo))
    x = torch.randn(batch, 1, hidden, generator=g).bfloat16()
    packed = linear(x.to(DEV), pq)
    y, size = oq.linear(x.view(batch, hidden), *wqkv)
    assert ((packed.view(batch, -1).cpu().double() - y).abs() <= oq.linear_bound(y, size, hidden)).all()
    cache = oq.random_cache(batch, hkv, capacity, dim, block, g)
    c = oq.to_device(cache, DEV)
    c = QuantCache(c["keys"], c["values"], c["key_scales"], c["value_scales"], block)
    ones = SimpleNamespace(weight=torch.ones(dim, dtype=torch.bfloat16, device=DEV), variance_epsilon=1e-6)
    cos, sin = torch.rand(capacity, dim, generator=g).bfloat16().to(DEV), torch.rand(capacity, dim, generator=g).bfloat16().to(DEV)
    query = qk_rope_cache_q8(packed, ones, ones, cos, sin, position.to(DEV), c, hq, rows=True,
                             phases=torch.zeros(batch, 1, dtype=torch.int64, device=DEV))
    at = position.clamp_min(0)
    heads = packed.cpu().double().view(batch, 1, hq + 2 * hkv, dim)
    turn = [t.cpu()[at][:, None, None] for t in (cos, sin)]
    gain = torch.ones(dim).bfloat16()
    expect = oq.norm_rope(heads[:, :, :hq], gain, 1e-6, *turn)
    noise = 2.0 ** -18 * expect.abs().amax(-1, keepdim=True)
    assert ((query.transpose(1, 2).cpu().double() - expect).abs() <= 2.0 ** -8 * expect.abs() + noise).all()
    after = {k: v.clone() if torch.is_tensor(v) else v for k, v in cache.items()}
    oq.append(after, "value", heads[:, :, hq + hkv:], position.tolist())
    assert torch.equal(c.values.cpu().view(torch.uint8), after["values"].view(torch.uint8))
    assert torch.equal(c.value_scales.cpu(), after["value_scales"])
    now = {"keys": c.keys.cpu(), "values": c.values.cpu(), "key_scales": c.key_scales.cpu(),
           "value_scales": c.value_scales.cpu(), "block": block}
    out = decode_attention_q8(query, c, position.to(DEV), 0.125)
    expect, bound = oq.attention(query.cpu().transpose(1, 2), now, position, 0.125)
    assert ((out.cpu().double() - expect).abs() <= bound).all() and (out[4] == 0).all()
    y, size = oq.linear(out.reshape(batch, -1).cpu(), *wo)
    last = linear(out.reshape(batch, 1, -1), po).view(batch, -1).cpu().double()
    assert ((last - y).abs() <= oq.linear_bound(y, size, hq * dim)).all()


def test_two_graphs_and_eager_calls_share_a_cache_handle():
    """Attention captured twice on one cache handle, replayed on two streams at once beside eager calls."""
    from kernels.decode_attention import decode_attention_q8
    g = torch.Generator(device=DEV).manual_seed(5)
    from kernels.quant import QuantCache
    codes = [(torch.randn(40, 8, 700, 128, device=DEV, generator=g) * 100).clamp(-448, 448).to(oq.E4M3) for _ in range(2)]
    scales = [torch.full((40, 8, 11), 2.0 ** -7, device=DEV) for _ in range(2)]
    cache = QuantCache(*codes, *scales, 64)
    position = torch.randint(0, 700, (40,), device=DEV, generator=g)
    queries = [torch.randn(40, 16, 1, 128, device=DEV, generator=g).bfloat16() for _ in range(3)]
    expect = [decode_attention_q8(q, cache, position, 0.09) for q in queries]
    streams, graphs, outs = [torch.cuda.Stream() for _ in range(2)], [], []
    torch.cuda.synchronize()
    for q, stream in zip(queries, streams):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            outs.append(decode_attention_q8(q, cache, position, 0.09))
        graphs.append(graph)
    for _ in range(20):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        third = decode_attention_q8(queries[2], cache, position, 0.09)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], expect[0]) and torch.equal(outs[1], expect[1]) and torch.equal(third, expect[2])


def test_append_then_attention_back_to_back():
    """Each append's slot is in the next attention, launched right behind it, over 40 steps."""
    from kernels.decode_attention import decode_attention_q8
    from kernels.qk_rope import qk_rope_cache_q8
    from kernels.quant import QuantCache
    g = torch.Generator().manual_seed(8)
    cache = QuantCache.zeros(2, 2, 64, 64, 16, DEV)
    one = SimpleNamespace(weight=torch.ones(64, dtype=torch.bfloat16, device=DEV), variance_epsilon=1e-6)
    cos, sin = torch.ones(1, 1, 64).bfloat16().to(DEV), torch.zeros(1, 1, 64).bfloat16().to(DEV)
    inputs = [(torch.randn(2, 1, 8 * 64, generator=g).bfloat16() * 2.0 ** (i % 5)).to(DEV) for i in range(40)]
    positions = [torch.tensor([i], device=DEV) for i in range(40)]
    outs = []
    for packed, position in zip(inputs, positions):
        query = qk_rope_cache_q8(packed, one, one, cos, sin, position, cache, 4)
        outs.append((query, decode_attention_q8(query, cache, position, 0.125)))
    # the same steps with a device synchronisation between the calls
    slow = QuantCache.zeros(2, 2, 64, 64, 16, DEV)
    for (query, out), packed, position in zip(outs, inputs, positions):
        again = qk_rope_cache_q8(packed, one, one, cos, sin, position, slow, 4)
        torch.cuda.synchronize()
        assert torch.equal(query, again)
        assert torch.equal(out, decode_attention_q8(again, slow, position, 0.125))
        torch.cuda.synchronize()
