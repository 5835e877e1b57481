"""DecodeState over the 8-bit cache and 4-bit weights: what a capture leaves behind."""

import pytest
import torch

import cases
import decode as fdecode
import qwen3

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(autouse=True)
def _no_device_errors():
    from kernels import _native
    _native.device_error()
    yield
    assert _native.device_error() == 0, "a kernel raised its device error word"


def tiny(group=0):
    cfg = qwen3.Config.make(**cases.TINY_QWEN3)
    weights = qwen3.from_state_dict(cfg, cases.tiny_qwen3_weights(), DEV)
    return qwen3.quantize_weights(weights, group) if group else weights


def state_of(weights, prompt, steps, block=16):
    return fdecode.DecodeState(weights, prompt.shape[0], prompt.shape[1], steps, kv_cache="q8", kv_block=block)


@pytest.mark.parametrize("block", [16, 32])
def test_capture_leaves_no_mark_in_the_cache(block):
    """A capture warms up with whatever token is in place; the step that follows may be given another
    (``step_host``). The warm-up's appends must not have raised a scale, nor rounded the codes under it once
    more: the replayed step equals an eager one on a state that was never captured."""
    prompt, _ = cases.model_prompt(cases.MODEL_CASES[1])  # 13 tokens: the next slot joins a block that holds some
    weights = tiny()
    length, token = prompt.shape[1], 77
    eager = state_of(weights, prompt, 6, block)
    eager.prefill(prompt.to(DEV))
    store, scales = eager.cache.store.clone(), eager.cache.scales.clone()
    eager.token_ids.fill_(token)
    eager.decode()
    for warm in range(5, 500, 33):
        state = state_of(weights, prompt, 6, block)
        state.prefill(prompt.to(DEV))
        state.token_ids.fill_(warm)
        state.capture()
        assert torch.equal(state.cache.scales, scales), warm
        assert torch.equal(state.cache.store[..., :length, :].view(torch.uint8), store[..., :length, :].view(torch.uint8))
        host_in = torch.full((prompt.shape[0],), token, dtype=torch.int64).pin_memory()
        host_out = torch.empty_like(host_in).pin_memory()
        state.step_host(host_in, host_out)
        torch.cuda.synchronize()
        state.release()
        assert torch.equal(host_out, eager.token_ids[:, 0].cpu())
        assert torch.equal(state.cache.scales, eager.cache.scales)
        for ours, theirs in zip(state.cache.layers, eager.cache.layers):
            for a, b in ((ours.keys, theirs.keys), (ours.values, theirs.values)):
                assert torch.equal(a[:, :, :length + 1].view(torch.uint8), b[:, :, :length + 1].view(torch.uint8))


# ------------------------------------------------------------------ tensor-parallel shards, one at a time
@pytest.mark.parametrize("form", ["push", "owner"])
@pytest.mark.parametrize("rows", [1, 16, 70])
def test_allreduce_of_a_4bit_projection_on_one_rank(form, rows):
    """The step's all-reduce after a 4-bit projection at world 1 (every region is this GPU's own): the projection
    comes finished, as one split, and the result is add + RMSNorm of it: the residual sum bit for bit."""
    import ctypes
    from types import SimpleNamespace
    from kernels.linear import linear
    from kernels.quant import quantize_weight4
    from kernels.rmsnorm import add_rms_norm
    g = torch.Generator().manual_seed(rows)
    n, k = 1024, 384
    weight = quantize_weight4((0.05 * torch.randn(n, k, generator=g)).bfloat16().to(DEV), 128)
    x = torch.randn(rows, 1, k, generator=g).bfloat16().to(DEV)
    residual = torch.randn(rows, 1, n, generator=g).bfloat16().to(DEV)
    gain = (1 + 0.1 * torch.randn(n, generator=g)).bfloat16().to(DEV)
    epoch = torch.full((1,), 9, dtype=torch.int64, device=DEV)
    shapes = {"recv": (2, 1, rows, n), "rs": (2, 1, rows, n), "ag": (2, rows, n // 2), "ss": (2, 1, n // 512, rows)}
    buffers = {name: torch.zeros(shape, dtype=torch.int64, device=DEV) for name, shape in shapes.items()}
    peers = SimpleNamespace(form=form, world=1)
    for name, buffer in buffers.items():
        setattr(peers, f"{name}_ptrs", (ctypes.c_void_p * 1)(buffer.data_ptr()))
        setattr(peers, f"{name}_local", ctypes.c_void_p(buffer.data_ptr()))
    out, summed = fdecode._allreduce_add_norm(x, weight, fdecode.Communicator(), peers, 1, epoch, residual, gain, 1e-6)
    torch.cuda.synchronize()
    expect, expect_sum = add_rms_norm(linear(x, weight), residual, gain, 1e-6)
    assert torch.equal(summed, expect_sum)
    # another order of the sum of squares: fp32 noise before two roundings to bf16
    assert ((out.float() - expect.float()).abs() <= 2.0 ** -7 * expect.float().abs() + 1e-30).all()


@pytest.mark.parametrize("world", [2])
def test_shards_are_slices_of_the_quantised_model(world):
    """Each rank quantises its shard; groups lie within the ranks' columns, so codes and scales are those of the
    whole model, and a rank's heads attend over its 8-bit cache as the whole model's do."""
    cfg = qwen3.Config.make(**cases.TINY_QWEN3)
    prompt, _ = cases.model_prompt(cases.MODEL_CASES[1])
    group, dim = 64, cfg.head_dim
    whole = qwen3.quantize_weights(qwen3.from_state_dict(cfg, cases.tiny_qwen3_weights(), DEV), group)
    hq, hkv, inter = cfg.num_attention_heads, cfg.num_key_value_heads, cfg.intermediate_size
    state = state_of(whole, prompt, 6)
    state.prefill(prompt.to(DEV))
    x = torch.randn(3, 1, cfg.hidden_size, generator=torch.Generator().manual_seed(2)).bfloat16().to(DEV)
    attended = state._rope_attention(x, whole.layers[0], 0)
    for rank in range(world):
        shard = qwen3.quantize_weights(qwen3.from_state_dict(cfg, cases.tiny_qwen3_weights(), DEV, rank, world), group)
        a, b = shard.layers[0], whole.layers[0]
        q, kv = slice(rank * hq // world, (rank + 1) * hq // world), slice(rank * hkv // world, (rank + 1) * hkv // world)
        heads = b.qkv.dequantized().view(hq + 2 * hkv, dim, -1)
        part = torch.cat((heads[:hq][q], heads[hq:hq + hkv][kv], heads[hq + hkv:][kv]))
        assert torch.equal(a.qkv.dequantized().view_as(part), part)
        assert torch.equal(a.o.dequantized(), b.o.dequantized()[:, q.start * dim:q.stop * dim])
        mlp = slice(rank * inter // world, (rank + 1) * inter // world)
        assert torch.equal(a.down.dequantized(), b.down.dequantized()[:, mlp])
        for ours, theirs in zip(qwen3.split_gate_up(a.gate_up.dequantized()), qwen3.split_gate_up(b.gate_up.dequantized())):
            assert torch.equal(ours, theirs[mlp])
        own = state_of(shard, prompt, 6)
        for ours, theirs in zip(own.cache.layers, state.cache.layers):
            for name in ("keys", "values", "key_scales", "value_scales"):
                getattr(ours, name).copy_(getattr(theirs, name)[:, kv])
        got = own._rope_attention(x, a, 0)
        for name in ("keys", "values", "key_scales", "value_scales"):  # the step appended the same slot
            ours, theirs = getattr(own.cache.layers[0], name), getattr(state.cache.layers[0], name)[:, kv]
            if name in ("keys", "values"):
                ours, theirs = ours.view(torch.uint8), theirs.view(torch.uint8)
            assert torch.equal(ours, theirs)
        # fewer units take another cluster size: fp32 sums in another order, one rounding to bf16 each
        expect = attended[:, :, q].float()
        assert ((got.float() - expect).abs() <= 2.0 ** -7 * expect.abs() + 2.0 ** -12 * expect.abs().amax()).all()
