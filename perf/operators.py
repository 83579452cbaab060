"""The attention layer of a decoder-type text model and products with 4-bit weights, as timed cases.

Three operators of ``iris_mi355x.kernels``, each at the sizes it is called with:

- ``rotary`` / ``rotary_store``: rotary positions in both layouts, over part of a head or all of it, with
  frequencies scaled for long contexts; K and V leaving for the caches that attention reads;
- ``window_attention``: attention with a sliding window and a few first tokens that stay visible, over
  whole prompts and for one or a few new tokens over a long cache;
- ``gemv_w4``: matrix-vector products with 4-bit weights and group scales.

Where ``own`` is false, ``run`` computes the same in elementary torch operations.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

HD = 128  # attention's head width


def _kernels():
    path = str(Path(__file__).resolve().parents[1] / "iris-3b-metal_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from iris_mi355x import kernels

    return kernels


def listed() -> list[dict]:
    return [
        # one new token of one sequence: q | k | v of a 2560-wide layer, K and V into the caches
        dict(name="rotary token", op="rotary", store=True, batch=1, tokens=1, heads=20, kv_heads=5, dim=128, part=128,
             layout="half", dtype="bf16", first=299, rows=512, scaling="none", transpose=False),
        # four prompts of 300 tokens, the text length of the denoiser, into their caches
        dict(name="rotary prompts", op="rotary", store=True, batch=4, tokens=300, heads=20, kv_heads=5, dim=128,
             part=128, layout="half", dtype="bf16", first=0, rows=512, scaling="none", transpose=False),
        # a long context at far positions: half of each head in interleaved pairs, frequencies by parts
        dict(name="rotary long", op="rotary", store=False, batch=1, tokens=32768, heads=32, kv_heads=8, dim=128, part=64,
             layout="interleaved", dtype="bf16", first=1000003, rows=0, scaling="by_parts", transpose=False),
        # the gradient of a batch of FP32 rows, an odd length
        dict(name="rotary gradient", op="rotary", store=False, batch=2, tokens=4097, heads=20, kv_heads=5, dim=128,
             part=128, layout="half", dtype="f32", first=0, rows=0, scaling="ntk", transpose=True),
        # one new token over a window of its cache
        dict(name="attention token", op="attention", batch=1, queries=1, keys=4096, heads=20, kv_heads=5, window=1024,
             sinks=4, causal=True, ragged=False, masked=False, token_major=False, fresh=False),
        # one new token of each of sixteen sequences of differing lengths, their whole caches
        dict(name="attention tokens long", op="attention", batch=16, queries=1, keys=65536, heads=32, kv_heads=8,
             window=0, sinks=0, causal=True, ragged=True, masked=False, token_major=False, fresh=False),
        # prompts padded on the left to 300 tokens: padding hidden by the mask, rows of padding see nothing
        dict(name="attention prompts", op="attention", batch=4, queries=300, keys=300, heads=20, kv_heads=5, window=128,
             sinks=4, causal=True, ragged=False, masked=True, token_major=True, fresh=True),
        # 256 text tokens that every image token sees, and a two-sided window over a megapixel's patches
        dict(name="attention joint", op="attention", batch=1, queries=4352, keys=4352, heads=20, kv_heads=5, window=640,
             sinks=256, causal=False, ragged=False, masked=False, token_major=True, fresh=True),
        # a long prompt
        dict(name="attention long", op="attention", batch=1, queries=8192, keys=8192, heads=32, kv_heads=8, window=4096,
             sinks=4, causal=True, ragged=False, masked=False, token_major=True, fresh=True),
        # the timestep MLP's square product, one row
        dict(name="w4 square", op="gemv", batch=1, n=2560, k=2560, group=64, zeros=False, dtype="f32", extra=0,
             silu=True),
        # the shared modulation core with every block's biases, a guidance batch
        dict(name="w4 core", op="gemv", batch=2, n=15360, k=2560, group=64, zeros=False, dtype="f32", extra=24,
             silu=True),
        # an MLP's first product for a batch of single tokens, zero points
        dict(name="w4 tokens", op="gemv", batch=24, n=13696, k=2560, group=128, zeros=True, dtype="bf16", extra=0,
             silu=False),
    ]


def _log_int(rng, low: int, high: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng) -> dict:
    op = rng.choice(["rotary", "attention", "attention", "gemv"])
    if op == "rotary":
        kv = rng.choice([1, 2, 5, 8])
        heads = kv * rng.choice([1, 2, 4, 7])
        dim = rng.choice([64, 80, 128, 256])
        part = rng.choice([dim, dim // 2, dim // 4])
        batch = _log_int(rng, 1, 16)
        tokens = _log_int(rng, 1, max(1, min(32768, 160_000_000 // (batch * (heads + 2 * kv) * dim))))
        store = rng.random() < 0.5
        first = rng.choice([0, 17, 4095, 1 << 20])
        return dict(op="rotary", store=store, batch=batch, tokens=tokens, heads=heads, kv_heads=kv, dim=dim, part=part,
                    layout=rng.choice(["half", "interleaved"]), dtype=rng.choice(["bf16", "f32"]), first=first,
                    rows=tokens + rng.randrange(40) if store else 0,
                    scaling=rng.choice(["none", "linear", "ntk", "by_parts"]),
                    transpose=not store and rng.random() < 0.3)
    if op == "attention":
        kv = rng.choice([1, 2, 5, 8])
        heads = kv * rng.choice([1, 2, 3, 4, 8])
        if rng.random() < 0.5:  # a few tokens over a cache
            queries = rng.choice([1, 1, 1, 2, 5])
            batch = _log_int(rng, 1, 16)
            keys = _log_int(rng, max(queries, 16), 65536)
            fresh = False
        else:
            batch = _log_int(rng, 1, 8)
            queries = _log_int(rng, 1, min(8192, int(math.sqrt(1.5e9 / (batch * heads)))))
            keys = queries
            fresh = True
        return dict(op="attention", batch=batch, queries=queries, keys=keys, heads=heads, kv_heads=kv,
                    window=rng.choice([0, _log_int(rng, 1, 4096)]), sinks=rng.choice([0, 1, 4, 77, 256]),
                    causal=not fresh or rng.random() < 0.6, ragged=not fresh and rng.random() < 0.6,
                    masked=rng.random() < 0.3, token_major=fresh or rng.random() < 0.3, fresh=fresh)
    group = rng.choice([32, 64, 128])
    k = 32 * _log_int(rng, 8, 428)
    n = _log_int(rng, 200, 27392)
    return dict(op="gemv", batch=_log_int(rng, 1, 64), n=n, k=k, group=group, zeros=rng.random() < 0.5,
                dtype=rng.choice(["f32", "bf16"]), extra=rng.choice([0, 0, 8]), silu=rng.random() < 0.4)


# ---------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------
def _dtype(case: dict) -> torch.dtype:
    return torch.float32 if case["dtype"] == "f32" else torch.bfloat16


def _randn(gen, *shape, dtype=torch.float32) -> torch.Tensor:
    return torch.randn(*shape, generator=gen, device="cuda").to(dtype)


def _frequencies(dim: int, scaling: str) -> tuple[torch.Tensor, float]:
    """Angles per position of the ``dim / 2`` pairs and the factor on the rotated values: contexts eight
    times the trained 4096 positions."""
    i = torch.arange(0, dim, 2, dtype=torch.float64) / dim
    theta, scale, trained = 10000.0, 8.0, 4096
    freqs = theta ** -i
    if scaling == "linear":
        return freqs / scale, 1.0
    if scaling == "ntk":
        return (theta * scale ** (dim / (dim - 2))) ** -i if dim > 2 else freqs, 1.0
    if scaling == "by_parts":  # pairs that turn often stay, pairs that turn less than once are stretched
        turns = trained * freqs / (2 * math.pi)
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0, 1)
        return freqs * keep + freqs / scale * (1 - keep), 0.1 * math.log(scale) + 1.0
    return freqs, 1.0


def _lengths(case: dict) -> list[int]:
    keys, batch = case["keys"], case["batch"]
    if not case["ragged"]:
        return [keys] * batch
    return [max(min(case["queries"], keys), keys - (b * keys) // (2 * batch)) for b in range(batch)]


def _padding(case: dict) -> list[int]:
    """Hidden keys at each sequence's front."""
    return [(b * case["keys"]) // (3 * case["batch"]) for b in range(case["batch"])] if case["masked"] else \
        [0] * case["batch"]


def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device="cuda").manual_seed(seed)
    state = dict(case)
    if case["op"] == "rotary":
        batch, tokens, heads, kv, dim = (case[key] for key in ("batch", "tokens", "heads", "kv_heads", "dim"))
        dtype = _dtype(case)
        proj = _randn(gen, batch, tokens, (heads + 2 * kv) * dim, dtype=dtype)  # a layer's packed projection
        state["q"] = proj[..., : heads * dim].view(batch, tokens, heads, dim)
        state["k"] = proj[..., heads * dim: (heads + kv) * dim].view(batch, tokens, kv, dim)
        state["v"] = proj[..., (heads + kv) * dim:].view(batch, tokens, kv, dim)
        freqs, state["factor"] = _frequencies(case["part"], case["scaling"])
        state["freqs"] = freqs.cuda()
        first = torch.arange(batch, device="cuda")[:, None] * 3 + case["first"]  # sequences at differing positions
        state["positions"] = first + torch.arange(tokens, device="cuda")
        if case["store"]:
            slots = torch.arange(batch, device="cuda")[:, None] % max(1, case["rows"] - tokens + 1)
            state["rows"] = slots + torch.arange(tokens, device="cuda")
            state["k_cache"] = _randn(gen, batch, kv, case["rows"], dim, dtype=dtype)
            state["v_cache"] = _randn(gen, batch, kv, case["rows"], dim, dtype=dtype)
    elif case["op"] == "attention":
        batch, nq, nk, heads, kv = (case[key] for key in ("batch", "queries", "keys", "heads", "kv_heads"))
        bf16 = torch.bfloat16

        def rows(h, n, token_major):
            if token_major:
                return _randn(gen, batch, n, h, HD, dtype=bf16).transpose(1, 2)
            return _randn(gen, batch, h, n, HD, dtype=bf16)

        if case["fresh"]:  # views of a prompt's packed projection
            proj = _randn(gen, batch, nq, heads + 2 * kv, HD, dtype=bf16).transpose(1, 2)
            state["q"], state["k"], state["v"] = proj[:, :heads], proj[:, heads:heads + kv], proj[:, heads + kv:]
        else:
            state["q"] = rows(heads, nq, True)
            state["k"], state["v"] = rows(kv, nk, case["token_major"]), rows(kv, nk, case["token_major"])
        state["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda") if case["ragged"] else None
        if case["masked"]:
            pad = torch.tensor(_padding(case), device="cuda")
            state["mask"] = torch.arange(nk, device="cuda")[None, :] >= pad[:, None]
        else:
            state["mask"] = None
        state["reach"] = case["window"] or None
    else:
        batch, n, k, group = case["batch"], case["n"], case["k"], case["group"]
        groups = -(-k // group)
        state["codes"] = torch.randint(0, 256, (n, k // 2), generator=gen, device="cuda", dtype=torch.uint8)
        spread = 1.0 + 0.3 * _randn(gen, n, groups)
        state["scales"] = (0.3 / math.sqrt(k) * spread).to(torch.bfloat16)
        state["zero_points"] = (torch.randint(4, 12, (n, groups), generator=gen, device="cuda", dtype=torch.uint8)
                                if case["zeros"] else None)
        state["x"] = _randn(gen, batch, k, dtype=_dtype(case))
        state["bias"] = 0.1 * _randn(gen, n)
        state["extra_bias"] = 0.1 * _randn(gen, case["extra"], n) if case["extra"] else None
        shape = (case["extra"], batch, n) if case["extra"] else (batch, n)
        state["out"] = torch.empty(shape, device="cuda", dtype=_dtype(case))
    return state


# ---------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------
def _rotate(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, layout: str) -> torch.Tensor:
    """``x`` ``[B, N, H, D]`` rotated by ``cos`` / ``sin`` ``[B, N, 1, P / 2]``, as ``[B, H, N, D]``."""
    part = 2 * cos.shape[-1]
    y = x.float()
    turned, rest = y[..., :part], y[..., part:]
    if layout == "half":
        a, b = turned[..., : part // 2], turned[..., part // 2:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    else:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    return torch.cat([turned, rest], dim=-1).to(x.dtype).transpose(1, 2).contiguous()


def _plain_rotary(s: dict):
    angles = s["positions"].double()[:, :, None, None] * s["freqs"]
    sign = -1.0 if s["transpose"] else 1.0
    cos, sin = (s["factor"] * angles.cos()).float(), (sign * s["factor"] * angles.sin()).float()
    q, k = _rotate(s["q"], cos, sin, s["layout"]), _rotate(s["k"], cos, sin, s["layout"])
    if not s["store"]:
        return q, k
    at = s["rows"][:, None, :, None].expand(-1, s["kv_heads"], -1, s["dim"])
    s["k_cache"].scatter_(2, at, k)
    s["v_cache"].scatter_(2, at, s["v"].transpose(1, 2))
    return q, s["k_cache"], s["v_cache"]


def _visible(s: dict) -> torch.Tensor:
    """``[B, Nq, Nk]``: which keys each query sees."""
    batch, nq, nk = s["batch"], s["queries"], s["keys"]
    j = torch.arange(nk, device="cuda")
    length = s["lengths"].long() if s["lengths"] is not None else torch.full((batch,), nk, device="cuda")
    p = (length - nq)[:, None, None] + torch.arange(nq, device="cuda")[:, None]
    seen = (j < length[:, None, None]).expand(-1, nq, -1)
    if s["causal"]:
        seen = seen & (j <= p)
    if s["window"]:
        seen = seen & (((p - j).abs() < s["window"]) | (j < s["sinks"]))
    if s["mask"] is not None:
        seen = seen & s["mask"][:, None, :]
    return seen


def _plain_attention(s: dict) -> torch.Tensor:
    batch, heads, nq, _ = s["q"].shape
    kv = s["kv_heads"]
    q = s["q"].float().reshape(batch, kv, heads // kv * nq, HD)
    k, v = s["k"].float().contiguous(), s["v"].float().contiguous()
    scores = (q @ k.transpose(-1, -2)).mul_(HD ** -0.5).view(batch, kv, heads // kv, nq, -1)
    scores.masked_fill_(~_visible(s)[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    weights = scores.sub_(torch.where(top.isfinite(), top, 0.0)).exp_()
    total = weights.sum(-1, keepdim=True)
    out = (weights.view(batch, kv, heads // kv * nq, -1) @ v).view(batch, kv, heads // kv, nq, HD)
    out = torch.where(total > 0, out / total, 0.0)
    return out.permute(0, 3, 1, 2, 4).reshape(batch, nq, heads * HD).to(torch.bfloat16)


def _plain_gemv(s: dict) -> torch.Tensor:
    codes = torch.stack([s["codes"] & 15, s["codes"] >> 4], dim=-1).flatten(1).float()
    zeros = 8.0 if s["zero_points"] is None else _per_weight(s["zero_points"].float(), s)
    weight = (codes - zeros) * _per_weight(s["scales"].float(), s)
    x = s["x"].float()
    if s["silu"]:
        x = x / (1.0 + torch.exp(-x))
    y = x @ weight.t() + s["bias"]
    if s["extra_bias"] is not None:
        y = y + s["extra_bias"][:, None, :]
    return y.to(s["x"].dtype)


def _per_weight(groups: torch.Tensor, s: dict) -> torch.Tensor:
    return groups.repeat_interleave(s["group"], dim=1)[:, : s["k"]]


def run(s: dict):
    if not own:
        return {"rotary": _plain_rotary, "attention": _plain_attention, "gemv": _plain_gemv}[s["op"]](s)
    K = _kernels()
    if s["op"] == "attention":
        return K.window_attention(s["q"], s["k"], s["v"], s["reach"], s["sinks"], causal=s["causal"],
                                  lengths=s["lengths"], key_mask=s["mask"])
    if s["op"] == "gemv":
        return K.gemv_w4(s["codes"], s["scales"], s["x"], s["bias"], s["out"], group=s["group"], zeros=s["zero_points"],
                         extra_bias=s["extra_bias"], in_silu=s["silu"])
    if s["store"]:
        q = K.rotary_store(s["q"], s["k"], s["v"], s["positions"], s["freqs"], s["k_cache"], s["v_cache"], s["rows"],
                           layout=s["layout"], factor=s["factor"])
        return q, s["k_cache"], s["v_cache"]
    return K.rotary(s["q"], s["k"], s["positions"], s["freqs"], layout=s["layout"], factor=s["factor"],
                    transpose=s["transpose"])


# ---------------------------------------------------------------------------------------
# what a pass costs, and its results in 64 bits
# ---------------------------------------------------------------------------------------
def _span(low: int, high: int, pad: int) -> tuple[int, int]:
    low = max(low, pad)
    return low, max(low, high)


def _pairs(case: dict) -> tuple[int, int]:
    """Visible (query, key) pairs of one head over the batch, and keys that some query sees."""
    pairs = seen = 0
    for length, pad in zip(_lengths(case), _padding(case)):
        reach, sinks = case["window"] or 1 << 40, case["sinks"] if case["window"] else 0
        first = length - case["queries"]
        spans = []
        for p in range(first, length):
            low, high = _span(max(0, p - reach + 1), min(length, p + 1 if case["causal"] else p + reach), pad)
            s_low, s_high = _span(0, min(sinks, low, p + 1 if case["causal"] else length), pad)
            pairs += high - low + s_high - s_low
            spans.append((low, high, s_low, s_high))
        band_low = min(x[0] for x in spans)
        band_high = max(max(x[1] for x in spans), band_low)
        sink = max(0, min(max(x[3] for x in spans), band_low) - min(x[2] for x in spans))
        seen += band_high - band_low + sink
    return pairs, seen


def work(case: dict) -> dict:
    if case["op"] == "rotary":
        rows = case["batch"] * case["tokens"]
        size = 4 if case["dtype"] == "f32" else 2
        heads = case["heads"] + case["kv_heads"] * (2 if case["store"] else 1)
        values = rows * heads * case["dim"]
        index = 8 * rows * (2 if case["store"] else 1)
        return {"bytes": 2 * values * size + index + 4 * case["part"],
                "flops": 3 * rows * (case["heads"] + case["kv_heads"]) * case["part"]}
    if case["op"] == "attention":
        pairs, seen = _pairs(case)
        rows = case["batch"] * case["queries"] * case["heads"]
        masks = case["batch"] * case["keys"] if case["masked"] else 0
        return {"bytes": 2 * 2 * rows * HD + 2 * 2 * seen * case["kv_heads"] * HD + masks,
                "flops": 4 * HD * pairs * case["heads"]}
    batch, n, k = case["batch"], case["n"], case["k"]
    groups = -(-k // case["group"])
    size = 4 if case["dtype"] == "f32" else 2
    extra = case["extra"]
    return {"bytes": n * k // 2 + n * groups * (3 if case["zeros"] else 2) + batch * k * size + 4 * n * (1 + extra)
            + batch * n * size * max(1, extra), "flops": 2 * batch * n * k}


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    if case["op"] == "rotary":
        angles = s["positions"].double().unsqueeze(-1) * s["freqs"]
        turn = torch.polar(torch.full_like(angles, s["factor"]), -angles if case["transpose"] else angles).unsqueeze(2)

        def rotated(x):
            x, part = x.double(), case["part"]
            if case["layout"] == "half":
                pairs = torch.complex(x[..., : part // 2].contiguous(), x[..., part // 2: part].contiguous()) * turn
                ends = torch.cat([pairs.real, pairs.imag], -1)
            else:
                pairs = torch.view_as_complex(x[..., :part].reshape(*x.shape[:-1], part // 2, 2)) * turn
                ends = torch.view_as_real(pairs).flatten(-2)
            return torch.cat([ends, x[..., part:]], -1).permute(0, 2, 1, 3)

        if not case["store"]:
            return rotated(s["q"]), rotated(s["k"])
        caches = s["k_cache"].double(), s["v_cache"].double()
        k, v = rotated(s["k"]), s["v"].double().permute(0, 2, 1, 3)
        item = torch.arange(case["batch"], device="cuda")[:, None]
        caches[0].transpose(1, 2)[item, s["rows"]] = k.transpose(1, 2)
        caches[1].transpose(1, 2)[item, s["rows"]] = v.transpose(1, 2)
        return rotated(s["q"]), *caches
    if case["op"] == "attention":
        if case["batch"] * case["heads"] * case["queries"] * case["keys"] > 3e9:
            return None
        group = case["heads"] // case["kv_heads"]
        out = torch.empty(case["batch"], case["queries"], case["heads"], HD, dtype=torch.float64, device="cuda")
        for b, (length, pad) in enumerate(zip(_lengths(case), _padding(case))):
            i = torch.arange(length - case["queries"], length, device="cuda").unsqueeze(1)
            j = torch.arange(pad, max(length, pad), device="cuda").unsqueeze(0)
            hidden = (j > i) if case["causal"] else torch.zeros_like(j > i)
            if case["window"]:
                far = (i - j >= case["window"]) | (j - i >= case["window"])
                hidden = hidden | (far & (j >= case["sinks"]))
            for h in range(case["heads"]):
                keys = s["k"][b, h // group, pad:max(length, pad)].double()
                values = s["v"][b, h // group, pad:max(length, pad)].double()
                logits = torch.mm(s["q"][b, h].double(), keys.t()) / math.sqrt(HD)
                weights = torch.softmax(logits.masked_fill(hidden, -math.inf), -1)
                out[b, :, h] = torch.mm(torch.where(hidden.all(-1, keepdim=True), 0.0, weights), values)
        return out.flatten(2)
    low, high = s["codes"].double() % 16, torch.div(s["codes"], 16, rounding_mode="floor").double()
    weight = torch.empty(case["n"], case["k"], dtype=torch.float64, device="cuda")
    weight[:, 0::2], weight[:, 1::2] = low, high
    of = torch.arange(case["k"], device="cuda") // case["group"]
    weight -= 8 if s["zero_points"] is None else s["zero_points"].double()[:, of]
    weight *= s["scales"].double()[:, of]
    x = s["x"].double()
    y = (x * torch.sigmoid(x) if case["silu"] else x) @ weight.t() + s["bias"].double()
    return y if s["extra_bias"] is None else y.unsqueeze(0) + s["extra_bias"].double().unsqueeze(1)
