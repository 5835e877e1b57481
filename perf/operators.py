"""Cases and plain forms of the quantised decode operators: attention over a KV cache held in 8
bits, the append that writes it, and projections with 4-bit weights.

``own`` selects what ``run`` calls: False, elementary torch operations in 32 bits; True, the
package's kernels through its public entry points. ``exact`` restates each operator in 64 bits.

The operators:

* ``decode`` / ``block``: one query token (or T of a verify block) per row over a cache of e4m3
  codes with one fp32 scale per (row, KV head, block of tokens), K and V apart.
* ``append``: per-head RMSNorm + rotate-half RoPE of a packed QKV projection; Q comes back, K and V
  are quantised into the cache. A block's scale is the least power of two that brings the largest
  magnitude of its valid slots to at most 448; a later token that needs a larger one has the
  block's earlier codes rounded once to it.
* ``linear``: y = x @ W^T, W = code * scale with 4-bit codes in [-8, 7] and one bf16 scale per row
  and group of columns.
"""

import math
import sys

import torch

own = False

DEV = "cuda"
PACKAGE = "fast-transformer_b200"  # holds the importable `kernels` package
E4M3_MAX = 448.0
EPS = 1e-6
LEAST_SCALE = 2.0 ** -100  # the scale of a block whose valid slots are all zero


def _package():
    if PACKAGE not in sys.path:
        sys.path.insert(0, PACKAGE)


# ------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one row of a 16/8-head model, 2048 cached tokens: the launch is what counts
        dict(name="decode-b1-l2048", op="decode", batch=1, q_heads=16, kv_heads=8, dim=128, capacity=2048, block=64,
             rows=False, least=2048),
        # a whole decode step's batch: 16 rows just past an 8192-token prompt
        dict(name="decode-b16-l8320", op="decode", batch=16, q_heads=32, kv_heads=8, dim=128, capacity=8320, block=64,
             rows=False, least=8320),
        # a serving batch of ragged rows, 1024 to 32768 tokens
        dict(name="decode-b64-ragged", op="decode", batch=64, q_heads=32, kv_heads=8, dim=128, capacity=32768, block=64,
             rows=True, least=1024),
        # head_dim 64, seven query heads a KV head, an odd capacity, rows with no token yet
        dict(name="decode-d64-odd", op="decode", batch=5, q_heads=14, kv_heads=2, dim=64, capacity=1003, block=16,
             rows=True, least=0),
        # a speculative verify pass: 5 tokens a row over 4096 cached ones
        dict(name="block-b8-t5", op="block", batch=8, q_heads=32, kv_heads=8, dim=128, capacity=4101, block=64,
             tokens=5, least=4101),
        # a long block (128 query members a KV head) over a short odd cache
        dict(name="block-b2-t16-d64", op="block", batch=2, q_heads=16, kv_heads=2, dim=64, capacity=777, block=32,
             tokens=16, least=300),
        # the append of one decode step, its newest token inside a block that has others
        dict(name="append-b16", op="append", batch=16, tokens=1, q_heads=32, kv_heads=8, dim=128, capacity=512,
             block=64, mode="decode", start=200),
        # a prompt of 8192 tokens written at once
        dict(name="append-prompt", op="append", batch=1, tokens=8192, q_heads=32, kv_heads=8, dim=128, capacity=8320,
             block=64, mode="prefill", start=0),
        # one row through a small model's projection: latency
        dict(name="linear-m1", op="linear", rows=1, n=4096, k=1024, group=64),
        # a batch of 16 through the wide MLP projection: the weight stream
        dict(name="linear-m16-wide", op="linear", rows=16, n=24576, k=4096, group=128),
        # a long, narrow product with small groups
        dict(name="linear-m5-long", op="linear", rows=5, n=4096, k=12288, group=32),
        # the widest batch that decodes together
        dict(name="linear-m64", op="linear", rows=64, n=6144, k=4096, group=128),
    ]


def _spread(rng, low, high):
    """A whole number in [low, high], spread over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["decode", "decode", "block", "append", "linear", "linear"])
    if op == "linear":
        group = rng.choice([32, 64, 128])
        rows, k = _spread(rng, 1, 64), _spread(rng, 2, 12288 // group) * group
        # no more than the widest listed product, nor more operations than the largest batch's
        most = min(24576, 24576 * 4096 // k, 64 * 6144 * 4096 // (rows * k))
        return dict(op=op, rows=rows, n=8 * _spread(rng, 8, max(8, most // 8)), k=k, group=group)
    dim, block = rng.choice([64, 128, 128]), rng.choice([16, 32, 64, 64])
    q_heads, kv_heads = rng.choice([(16, 8), (32, 8), (8, 1), (4, 4), (14, 2), (6, 2)])
    if op == "append":
        mode = rng.choice(["decode", "rows", "prefill"])
        tokens = {"decode": 1, "rows": _spread(rng, 1, 16), "prefill": _spread(rng, 2, 4096)}[mode]
        start = 0 if mode == "prefill" else _spread(rng, 1, 400)
        return dict(op=op, batch=_spread(rng, 1, 2 if mode == "prefill" else 48), tokens=tokens, q_heads=q_heads,
                    kv_heads=kv_heads, dim=dim, capacity=start + tokens + _spread(rng, 1, 200), block=block, mode=mode,
                    start=start)
    batch = _spread(rng, 1, 64 if op == "decode" else 16)
    capacity = _spread(rng, 48, min(32768, 64 * 8 * 8192 // (batch * kv_heads)))
    case = dict(op=op, batch=batch, q_heads=q_heads, kv_heads=kv_heads, dim=dim, capacity=capacity, block=block)
    if op == "decode":
        rows = rng.random() < 0.6
        return dict(case, rows=rows, least=rng.choice([0, capacity // 3]) if rows else capacity)
    return dict(case, tokens=rng.randint(2, 16), least=rng.choice([32, max(32, capacity // 2)]))


# ------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    state = {"case": case}
    if case["op"] == "linear":
        n, k, group = case["n"], case["k"], case["group"]
        state["x"] = torch.randn(case["rows"], k, device=DEV, generator=g).bfloat16()
        state["codes"] = torch.randint(-8, 8, (n, k), device=DEV, generator=g, dtype=torch.int8)
        state["scales"] = (0.004 + 0.004 * torch.rand(n, k // group, device=DEV, generator=g)).bfloat16()
        if own:  # the weights are laid out once, as a program that loads them does
            _package()
            from kernels.quant import pack_weight4
            state["weight"] = pack_weight4(state["codes"], state["scales"])
        return state
    batch, q_heads, kv_heads, dim = case["batch"], case["q_heads"], case["kv_heads"], case["dim"]
    capacity, block = case["capacity"], case["block"]

    def cache(least, most):
        # codes as a scaled block holds them, and scales of neighbouring magnitudes
        codes = torch.empty(batch, kv_heads, capacity, dim, device=DEV, dtype=torch.float8_e4m3fn)
        for row in range(batch):
            part = torch.randn(kv_heads, capacity, dim, device=DEV, generator=g)
            codes[row].copy_((part * 112.0).clamp_(-E4M3_MAX, E4M3_MAX))
        exponents = torch.randint(least, most + 1, (batch, kv_heads, -(-capacity // block)), device=DEV, generator=g)
        return codes, torch.exp2(exponents.float())

    state["keys"], state["key_scales"] = cache(-8, -6)
    state["values"], state["value_scales"] = cache(-9, -7)
    if own:  # the handle that a decoding program keeps for a layer's cache
        _package()
        from kernels.quant import QuantCache
        state["cache"] = QuantCache(state["keys"], state["values"], state["key_scales"], state["value_scales"], block)
    if case["op"] == "append":
        tokens, start = case["tokens"], case["start"]
        width = (q_heads + 2 * kv_heads) * dim
        state["packed"] = torch.randn(batch, tokens, width, device=DEV, generator=g).bfloat16()
        state["q_weight"] = (1 + 0.1 * torch.randn(dim, device=DEV, generator=g)).bfloat16()
        state["k_weight"] = (1 + 0.1 * torch.randn(dim, device=DEV, generator=g)).bfloat16()
        rows = case["mode"] == "rows"
        if rows:
            position = torch.randint(0, start + 1, (batch,), device=DEV, generator=g)
            places = position[:, None] + torch.arange(tokens, device=DEV)
        else:
            position = torch.arange(tokens, device=DEV) if case["mode"] == "prefill" else torch.tensor([start], device=DEV)
            places = start + torch.arange(tokens, device=DEV)[None]
        angles = places[..., None].double() * 1e6 ** (-torch.arange(0, dim, 2, device=DEV).double() / dim)
        angles = torch.cat((angles, angles), -1)
        state["cos"], state["sin"] = angles.cos().bfloat16().contiguous(), angles.sin().bfloat16().contiguous()
        state["position"] = position
        if own:
            state["q_norm"], state["k_norm"] = _Norm(state["q_weight"]), _Norm(state["k_weight"])
        return state
    tokens = case.get("tokens", 1)
    state["scale"] = 1.0 / math.sqrt(dim)
    if case["op"] == "decode":
        state["query"] = torch.randn(batch, q_heads, 1, dim, device=DEV, generator=g).bfloat16()
        if case["rows"]:  # lengths from `least` to the capacity; position -1 is a row without a token
            lengths = torch.randint(case["least"], capacity + 1, (batch,), device=DEV, generator=g)
            state["position"] = lengths - 1
        else:
            state["position"] = torch.tensor([capacity - 1], device=DEV)
        return state
    state["query"] = torch.randn(batch, tokens, q_heads, dim, device=DEV, generator=g).bfloat16()
    least = min(case["least"], capacity)
    lengths = torch.randint(max(least, tokens), capacity + 1, (batch,), device=DEV, generator=g)
    state["position"] = lengths - tokens
    state["chain"] = torch.randint(1, tokens + 1, (batch,), device=DEV, generator=g)
    return state


class _Norm:
    """The gain and epsilon of a head norm, as the append's entry point reads them."""

    def __init__(self, weight):
        self.weight, self.variance_epsilon = weight, EPS


# --------------------------------------------------------------------------------- plain forms
def _values(codes, scales, block):
    """What a cache's codes stand for, in 32 bits."""
    capacity = codes.shape[2]
    return codes.float() * scales.repeat_interleave(block, 2)[:, :, :capacity, None]


def _visible(case, position, chain):
    """[B, T, C]: which cache slots each token of each row attends to."""
    slots = torch.arange(case["capacity"], device=DEV)
    if chain is None:
        return (slots <= position[:, None, None]).expand(case["batch"], 1, -1)
    token = torch.arange(case["tokens"], device=DEV)
    own_slot = position[:, None] + token
    last = torch.where(token < chain[:, None], own_slot, position[:, None])
    return (slots <= last[..., None]) | (slots == own_slot[..., None])


def _attention(case, query, keys, values, visible, scale):
    """query [B, T, Hq, D]; keys, values [B, Hkv, C, D] -> [B, T, Hq, D], all in one type."""
    batch, tokens, q_heads, dim = query.shape
    kv_heads = keys.shape[1]
    groups = q_heads // kv_heads
    members = query.reshape(batch, tokens, kv_heads, groups, dim).permute(0, 2, 1, 3, 4)
    members = members.reshape(batch, kv_heads, tokens * groups, dim)
    scores = torch.matmul(members, keys.transpose(2, 3)) * scale
    seen = visible[:, None, :, None].expand(batch, kv_heads, tokens, groups, -1).reshape(scores.shape)
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    weights = (scores - torch.where(top == -math.inf, 0.0, top)).exp()
    total = weights.sum(-1, keepdim=True)
    out = torch.matmul(weights, values) / torch.where(total == 0, 1.0, total)
    out = out.reshape(batch, kv_heads, tokens, groups, dim).permute(0, 2, 1, 3, 4)
    return out.reshape(batch, tokens, q_heads, dim)


def _norm_rope(x, weight, cos, sin):
    """x [B, T, H, D] in 32 or 64 bits; cos, sin [B or 1, T, D]."""
    normed = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight.to(x.dtype)
    half = x.shape[-1] // 2
    turned = torch.cat((-normed[..., half:], normed[..., :half]), -1)
    return normed * cos.to(x.dtype)[:, :, None] + turned * sin.to(x.dtype)[:, :, None]


def _least_scale(largest):
    """The least power of two s with largest <= 448 s."""
    fraction, exponent = torch.frexp(largest)
    s = torch.exp2((exponent - torch.where(fraction <= 0.875, 9, 8)).to(largest.dtype))
    return torch.where(largest > 0, s, torch.zeros_like(s)).clamp_min(LEAST_SCALE)


def _append(case, codes, scales, new, start, round_codes):
    """Writes `new` [B, T, H, D] at slots start[b] + t: (touched slots, their codes in `new`'s type,
    the touched blocks, their scales, which touched slots hold something)."""
    batch, tokens, heads, dim = new.shape
    block, capacity = case["block"], case["capacity"]
    blocks = (tokens + block - 2) // block + 1
    first = start // block  # [B]
    slots = first[:, None] * block + torch.arange(blocks * block, device=DEV)
    token = slots - start[:, None]
    fresh, earlier = (token >= 0) & (token < tokens), token < 0
    at = torch.where(slots < capacity, slots, start[:, None])  # past the cache: the first new slot again
    index = at[:, None, :, None].expand(batch, heads, -1, dim)
    old = codes.view(torch.uint8).gather(2, index).view(torch.float8_e4m3fn).to(new.dtype)
    which = at - start[:, None]
    x = new.permute(0, 2, 1, 3).gather(2, which.clamp(0, tokens - 1)[:, None, :, None].expand(batch, heads, -1, dim))
    sizes = (x.abs() * fresh[:, None, :, None]).reshape(batch, heads, blocks, block * dim)
    place = (first[:, None] + torch.arange(blocks, device=DEV)).clamp_max(scales.shape[2] - 1)
    place = place[:, None].expand(batch, heads, -1)
    before = scales.gather(2, place).to(new.dtype)
    holds = earlier.reshape(batch, 1, blocks, block).any(-1)
    wanted = _least_scale(sizes.amax(-1))
    after = torch.where(holds, torch.maximum(wanted, before), wanted)
    touched = fresh.reshape(batch, 1, blocks, block).any(-1)
    after = torch.where(touched, after, before)
    of = (at // block - first[:, None])[:, None].expand(batch, heads, -1)  # each slot's touched block
    per_slot, ratio = after.gather(2, of)[..., None], (before / after).gather(2, of)[..., None]
    kept = torch.where(earlier[:, None, :, None], old * ratio, old)  # slots behind the new ones stay as they are
    held = ((which >= 0) & (which < tokens))[:, None, :, None]
    result = torch.where(held, round_codes(x / per_slot), round_codes(kept))
    return index, result, place, after, touched.expand_as(after)


def _e4m3(x):
    return x.to(torch.float8_e4m3fn)


def _write(codes, scales, index, result, place, after, touched):
    codes.view(torch.uint8).scatter_(2, index, result.view(torch.uint8))
    # blocks that got no token leave their scale; a repeated last block must not win over it
    held = torch.where(touched, after, torch.zeros_like(after))
    fresh = torch.zeros_like(scales).scatter_reduce_(2, place, held, "amax")
    scales.copy_(torch.where(fresh > 0, fresh, scales))


def _split_packed(case, packed):
    batch, tokens, dim = case["batch"], case["tokens"], case["dim"]
    hq, hkv = case["q_heads"], case["kv_heads"]
    heads = packed.reshape(batch, tokens, hq + 2 * hkv, dim)
    return heads[:, :, :hq], heads[:, :, hq:hq + hkv], heads[:, :, hq + hkv:]


def _starts(case, position):
    if case["mode"] == "rows":
        return position
    return torch.full((case["batch"],), case["start"], device=DEV, dtype=torch.int64)


def run(state):
    case = state["case"]
    op = case["op"]
    if op == "linear":
        if own:
            from kernels.linear import linear
            return linear(state["x"], state["weight"])
        weight = state["codes"].float() * state["scales"].float().repeat_interleave(case["group"], 1)
        return torch.matmul(state["x"].float(), weight.t()).bfloat16()
    if op == "append":
        if own:
            from kernels.qk_rope import qk_rope_cache_q8
            query = qk_rope_cache_q8(state["packed"], state["q_norm"], state["k_norm"], state["cos"], state["sin"],
                                     state["position"], state["cache"], case["q_heads"],
                                     prefill=case["mode"] == "prefill", rows=case["mode"] == "rows")
            query = query.transpose(1, 2)
        else:
            q, k, v = _split_packed(case, state["packed"].float())
            query = _norm_rope(q, state["q_weight"], state["cos"], state["sin"]).bfloat16()
            k = _norm_rope(k, state["k_weight"], state["cos"], state["sin"])
            start = _starts(case, state["position"])
            _write(state["keys"], state["key_scales"], *_append(case, state["keys"], state["key_scales"], k, start, _e4m3))
            _write(state["values"], state["value_scales"],
                   *_append(case, state["values"], state["value_scales"], v, start, _e4m3))
        return {"query": query, "keys": state["keys"], "values": state["values"], "key_scales": state["key_scales"],
                "value_scales": state["value_scales"]}
    if own:
        from kernels.decode_attention import block_attention_q8, decode_attention_q8
        if op == "decode":
            return decode_attention_q8(state["query"], state["cache"], state["position"], state["scale"])
        return block_attention_q8(state["query"], state["cache"], state["position"], state["scale"], state["chain"])
    query = state["query"].float()
    query = query.transpose(1, 2) if op == "decode" else query
    out = _attention(case, query, _values(state["keys"], state["key_scales"], case["block"]),
                     _values(state["values"], state["value_scales"], case["block"]),
                     _visible(case, state["position"], state.get("chain")), state["scale"])
    return out.bfloat16()


# ---------------------------------------------------------------------------------------- work
def work(case):
    op = case["op"]
    if op == "linear":
        rows, n, k = case["rows"], case["n"], case["k"]
        return {"bytes": n * k / 2 + n * (k // case["group"]) * 2 + rows * (n + k) * 2, "flops": 2 * rows * n * k}
    batch, hq, hkv, dim = case["batch"], case["q_heads"], case["kv_heads"], case["dim"]
    if op == "append":
        tokens = case["tokens"]
        q, kv = batch * tokens * hq * dim, batch * tokens * hkv * dim
        scales = 2 * batch * hkv * (-(-tokens // case["block"])) * 4
        return {"bytes": 2 * q + 2 * 2 * kv + 2 * q + 2 * kv + scales + 2 * tokens * dim * 2, "flops": 10 * (q + 2 * kv)}
    tokens = case.get("tokens", 1)
    # lengths are drawn evenly between the least and the capacity
    slots = batch * hkv * (min(case["least"], case["capacity"]) + case["capacity"]) / 2
    members = tokens * hq // hkv
    return {"bytes": 2 * slots * (dim + 4 / case["block"]) + 2 * 2 * batch * tokens * hq * dim,
            "flops": 4 * slots * members * dim}


# --------------------------------------------------------------------------------------- exact
def exact(case, seed):
    """The operators restated in 64 bits: rows one at a time, masks by slicing."""
    state = prepare(case, seed)
    op = case["op"]
    if op == "linear":
        n, k, group = case["n"], case["k"], case["group"]
        x = state["x"].double()
        out = torch.zeros(case["rows"], n, device=DEV, dtype=torch.float64)
        for low in range(0, n, 4096):
            part = state["codes"][low:low + 4096].double().reshape(-1, k // group, group)
            part = part * state["scales"][low:low + 4096].double()[:, :, None]
            out[:, low:low + 4096] = x @ part.reshape(-1, k).t()
        return out
    block = case["block"]
    if op == "append":
        return _exact_append(case, state)
    query = state["query"].double()
    query = query.transpose(1, 2) if op == "decode" else query
    batch, tokens, q_heads, dim = query.shape
    kv_heads = case["kv_heads"]
    groups = q_heads // kv_heads
    out = torch.zeros(batch, tokens, q_heads, dim, device=DEV, dtype=torch.float64)
    position = state["position"].expand(batch).tolist()
    chain = state["chain"].tolist() if "chain" in state else [1] * batch
    for b in range(batch):
        for t in range(tokens):
            seen = position[b] + 1 + (t if t < chain[b] else 0)
            if seen <= 0:
                continue
            index = torch.arange(seen, device=DEV)
            if t >= chain[b]:
                index = torch.cat((index, index.new_tensor([position[b] + t])))
            keys = state["keys"][b].view(torch.uint8)[:, index].view(torch.float8_e4m3fn).double()
            keys = keys * state["key_scales"][b][:, index // block, None].double()
            vals = state["values"][b].view(torch.uint8)[:, index].view(torch.float8_e4m3fn).double()
            vals = vals * state["value_scales"][b][:, index // block, None].double()
            scores = torch.einsum("hgd,hcd->hgc", query[b, t].reshape(kv_heads, groups, dim), keys) * state["scale"]
            weights = torch.softmax(scores, -1)
            out[b, t] = torch.einsum("hgc,hcd->hgd", weights, vals).reshape(q_heads, dim)
    return out


def _exact_append(case, state):
    batch, tokens, dim, block = case["batch"], case["tokens"], case["dim"], case["block"]
    hq, hkv = case["q_heads"], case["kv_heads"]
    heads = state["packed"].double().reshape(batch, tokens, hq + 2 * hkv, dim)
    cos, sin = (state[n].double().expand(batch, tokens, dim)[:, :, None] for n in ("cos", "sin"))

    def turn(x, gain):
        x = x / (x.pow(2).sum(-1, keepdim=True) / dim + EPS).sqrt() * gain.double()
        low, high = x.chunk(2, -1)
        return x * cos + torch.cat((-high, low), -1) * sin

    query = turn(heads[:, :, :hq], state["q_weight"])
    result = {"query": query}
    new = {"key": turn(heads[:, :, hq:hq + hkv], state["k_weight"]), "value": heads[:, :, hq + hkv:]}
    starts = state["position"].tolist() if case["mode"] == "rows" else [case["start"]] * batch
    for name, x in new.items():
        codes, scales = state[name + "s"].double(), state[name + "_scales"].double()
        for b in range(batch):
            for at in range(starts[b] // block, (starts[b] + tokens - 1) // block + 1):
                low = max(starts[b], at * block)
                high = min(starts[b] + tokens, (at + 1) * block)
                part = x[b, low - starts[b]:high - starts[b]].transpose(0, 1)  # [H, slots, D]
                largest = part.abs().amax((1, 2)).clamp_min(1e-300)
                need = torch.exp2(torch.ceil(torch.log2(largest / E4M3_MAX))).clamp_min(LEAST_SCALE)
                if low > at * block:
                    need = torch.maximum(need, scales[b, :, at])
                    codes[b, :, at * block:low] *= (scales[b, :, at] / need)[:, None, None]
                codes[b, :, low:high] = part / need[:, None, None]
                scales[b, :, at] = need
        result[name + "s"], result[name + "_scales"] = codes, scales
    return result
