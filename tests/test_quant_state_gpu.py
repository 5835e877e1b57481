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
