"""The quantised decode operators in 64 bits: attention over the 8-bit cache, the append that
writes it, the move of a slot, and 4-bit projections. Restated from their definitions (they have
no counterpart in the reference), with the error bounds that the rounding of each allows.

A cache is a dict: ``keys``, ``values`` (torch.float8_e4m3fn [B, Hkv, C, D]), ``key_scales``,
``value_scales`` (fp32 [B, Hkv, ceil(C / block)]) and ``block``.
"""

import math

import torch

E4M3 = torch.float8_e4m3fn
LEAST_SCALE = 2.0 ** -100


def empty_cache(batch, kv_heads, capacity, dim, block):
    scales = (batch, kv_heads, -(-capacity // block))
    return {"keys": torch.zeros(batch, kv_heads, capacity, dim).to(E4M3),
            "values": torch.zeros(batch, kv_heads, capacity, dim).to(E4M3),
            "key_scales": torch.zeros(scales), "value_scales": torch.zeros(scales), "block": block}


def random_cache(batch, kv_heads, capacity, dim, block, generator):
    """Codes as scaled blocks hold them and power-of-two scales of neighbouring magnitudes."""
    def codes():
        x = torch.randn(batch, kv_heads, capacity, dim, generator=generator) * 112.0
        return x.clamp(-448.0, 448.0).to(E4M3)

    def scales(low, high):
        e = torch.randint(low, high + 1, (batch, kv_heads, -(-capacity // block)), generator=generator)
        return torch.exp2(e.float())

    return {"keys": codes(), "values": codes(), "key_scales": scales(-8, -6), "value_scales": scales(-9, -7),
            "block": block}


def to_device(cache, device):
    return {k: v.to(device) if torch.is_tensor(v) else v for k, v in cache.items()}


def visible(position, tokens, chain, t, capacity):
    """Slots token t of a row sees (position: the row's first token's slot; chain None: decode)."""
    if position < 0:
        return torch.zeros(0, dtype=torch.int64)
    last = position + (t if chain is not None and t < chain else 0)
    slots = list(range(0, min(last + 1, capacity)))
    if chain is not None and t >= chain and position + t < capacity:
        slots.append(position + t)
    return torch.tensor(slots, dtype=torch.int64)


def attention(query, cache, position, scale, chain=None):
    """query [B, T, Hq, D] -> (out, bound) in 64 bits. ``bound``: how far a bf16 result may be off that
    sums in fp32 and rounds P (scaled by V's block scale against its largest) to f16:
      2^-8 |out|  (the output) + sum_c max(2^-11 p'_c, 2^-32 p'_top) |vcode_c|
      (P: 2^-11 of a normal f16, 2^-25 of a subnormal one, the largest weight being held at 2^7 or above)
      + eps * sum_c p_c |v_c|,  eps = the scores' and the sums' fp32 rounding."""
    batch, tokens, q_heads, dim = query.shape
    kv_heads, capacity = cache["keys"].shape[1:3]
    groups, block = q_heads // kv_heads, cache["block"]
    out = torch.zeros(batch, tokens, q_heads, dim, dtype=torch.float64)
    bound = torch.zeros_like(out)
    for b in range(batch):
        for t in range(tokens):
            at = visible(int(position[b if len(position) > 1 else 0]), tokens, None if chain is None else int(chain[b]),
                         t, capacity)
            if len(at) == 0:
                continue
            ks = cache["key_scales"][b][:, at // block].double()
            vs = cache["value_scales"][b][:, at // block].double()
            k = cache["keys"][b].float()[:, at].double() * ks[..., None]
            codes = cache["values"][b].float()[:, at].double()
            q = query[b, t].double().reshape(kv_heads, groups, dim)
            scores = torch.einsum("hgd,hcd->hgc", q, k) * scale
            p = torch.softmax(scores, -1)
            v = codes * vs[..., None]
            out[b, t] = torch.einsum("hgc,hcd->hgd", p, v).reshape(q_heads, dim)
            size = torch.einsum("hgc,hcd->hgd", p, v.abs())
            weight = p * vs[:, None]
            top = weight.amax(-1, keepdim=True).clamp_min(1e-300)
            rounding = torch.maximum(2.0 ** -11 * weight, 2.0 ** -32 * (1 + 2.0 ** -16) * top)  # 2^7 to fp32's rounding
            by_p = torch.einsum("hgc,hcd->hgd", rounding, codes.abs())
            largest = torch.einsum("hgd,hcd->hgc", q.abs(), k.abs()).amax() * abs(scale)
            eps = float(largest) * 4 * dim * 2.0 ** -23 + (len(at) / 16 + 64) * 2.0 ** -23 + 2.0 ** -20
            bound[b, t] = (2.0 ** -8 * out[b, t].abs().reshape(kv_heads, groups, dim) + by_p + eps * size).reshape(
                q_heads, dim)
    return out, bound


def norm_rope(x, gain, eps, cos, sin):
    """x [..., D] in 64 bits; cos, sin [..., D] of the token's phase."""
    w = x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt() * gain.double()
    low, high = w.chunk(2, -1)
    return w * cos.double() + torch.cat((-high, low), -1) * sin.double()


def least_scale(largest):
    if largest <= 448.0 * LEAST_SCALE:
        return LEAST_SCALE
    scale = 2.0 ** math.floor(math.log2(largest / 448.0))
    while scale * 448.0 < largest:
        scale *= 2.0
    return scale


def append(cache, name, new, starts):
    """Writes new [B, T, Hkv, D] (64 bits) at slots starts[b] + t of ``name`` ("key" or "value") in
    place; returns the unrounded values [B, Hkv, C, D] of every slot (earlier slots: their codes
    before the call times their scale)."""
    codes, scales, block = cache[name + "s"], cache[name + "_scales"], cache["block"]
    batch, tokens, heads, dim = new.shape
    capacity = codes.shape[2]
    real = codes.double() * scales.double().repeat_interleave(block, 2)[:, :, :capacity, None]
    for b in range(batch):
        start = int(starts[b])
        if start < 0:
            continue
        end = min(start + tokens, capacity)
        for at in range(start // block, (end - 1) // block + 1):
            low, high = max(start, at * block), min(end, (at + 1) * block)
            for h in range(heads):
                part = new[b, low - start:high - start, h]
                finite = part[torch.isfinite(part)].abs()
                scale = least_scale(float(finite.max()) if finite.numel() else 0.0)
                if low > at * block:
                    before = float(scales[b, h, at])
                    scale = max(scale, before)
                    old = codes[b, h, at * block:low].float() * (before / scale)
                    codes[b, h, at * block:low] = old.to(E4M3)
                real[b, h, low:high] = part
                scaled = (part / scale).float()
                codes[b, h, low:high] = torch.where(torch.isfinite(scaled), scaled, float("nan")).to(E4M3)
                scales[b, h, at] = scale
    return real


def relocate(codes, scales, block, move_from, move_to):
    """codes [P, B, H, C, D] (P = planes x layers), scales [P, B, H, blocks], in place."""
    planes, batch, heads = codes.shape[:3]
    for b in range(batch):
        source, target = int(move_from[b]), int(move_to[b])
        if source < 0:
            continue
        for i in range(planes):
            for h in range(heads):
                c, s = codes[i, b, h], scales[i, b, h]
                if source // block == target // block:
                    c.view(torch.uint8)[target] = c.view(torch.uint8)[source]
                    continue
                value = c[source].float() * s[source // block]
                finite = value[torch.isfinite(value)].abs()
                scale = least_scale(float(finite.max()) if finite.numel() else 0.0)
                low = target // block * block
                if target > low:
                    before = float(s[target // block])
                    scale = max(scale, before)
                    c[low:target] = (c[low:target].float() * (before / scale)).to(E4M3)
                c[target] = (value / scale).to(E4M3)
                s[target // block] = scale


def linear(x, codes, scales):
    """(y, size): x [M, K] @ W^T in 64 bits and sum |x| |w|, W = codes * scales per row and group."""
    n, k = codes.shape
    w = codes.double() * scales.double().repeat_interleave(k // scales.shape[1], 1)
    return x.double() @ w.t(), x.double().abs() @ w.abs().t()


def linear_bound(y, size, k, rounded=True):
    """fp32 sums in tensor-core products of 16 columns, chains of 4, then at most k / 64 totals and 16
    partial sums (each at most one step of 2^-23), and one rounding to bf16."""
    return (2.0 ** -8 * y.abs() if rounded else 0) + (24 + k / 64 + 16) * 2.0 ** -23 * size
