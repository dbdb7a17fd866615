"""The cache-maintenance operators of one layer's packed KV cache, as measured cases.

Around the decode attention over packed INT2/INT4 blocks a serving loop needs four more things:

* ``rotary``: rotary positions of query (or key) heads, half or interleaved pairs, on part of the
  head, with frequencies scaled for long contexts;
* ``append``: the new tokens' keys (rotated) and values quantized into their slots of the block
  pool, with the FP16 values the cache now holds for them;
* ``weights``: the attention weight each cached token gets, summed over the query heads of its KV
  head and over the queries, added to what it got before;
* ``evict``: from those sums the tokens each KV head keeps, and the cache compacted to them.

A case is one call of one of them. ``run`` computes it with elementary torch operations, or, where
``own`` is true, with ``kvssd_b200.ops``.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # One decode step's query heads of 8 sequences, about a million tokens into a context: the
        # call that latency decides.
        dict(name="rotary_step", op="rotary", tokens=8, heads=32, dim=128, part=128, dtype="f16",
             interleaved=False, scaling="smooth", far=1048576, strided=False),
        # The query heads of an 8192-token prompt, cut out of a fused projection's output.
        dict(name="rotary_prompt", op="rotary", tokens=8192, heads=32, dim=128, part=128,
             dtype="bf16", interleaved=False, scaling="yarn", far=8192, strided=True),
        # Interleaved pairs on half of a 64-wide head in FP32, odd length.
        dict(name="rotary_part", op="rotary", tokens=4099, heads=24, dim=64, part=32, dtype="f32",
             interleaved=True, scaling="linear", far=131072, strided=False),
        # One decode step of 16 sequences (one of them padding) over a shared pool.
        dict(name="append_step", op="append", tokens=16, kv_heads=8, dim=128, bits=4, group=32,
             block=128, blocks=1024, part=128, dtype="f16", interleaved=False, far=131072,
             holes=1, outliers=0.0),
        # An 8192-token prompt into 64 fresh blocks.
        dict(name="append_prompt", op="append", tokens=8192, kv_heads=8, dim=128, bits=4, group=32,
             block=128, blocks=64, part=128, dtype="bf16", interleaved=False, far=8192, holes=0,
             outliers=0.0),
        # A longer ragged prompt chunk with outlier channels into an INT2 cache, partial rotary.
        dict(name="append_int2", op="append", tokens=16411, kv_heads=8, dim=128, bits=2, group=32,
             block=128, blocks=160, part=64, dtype="f16", interleaved=True, far=131072, holes=3,
             outliers=0.01),
        # One decode step's weights over 8192 tokens: the attention's log-sum-exp is at hand.
        dict(name="weights_step", op="weights", queries=1, heads=32, kv_heads=8, dim=128, bits=4,
             group=32, block=128, tokens=8192, dtype="f16", table=False, lse=True, seen="all"),
        # The same over 131072 tokens.
        dict(name="weights_step_128k", op="weights", queries=1, heads=32, kv_heads=8, dim=128,
             bits=4, group=32, block=128, tokens=131072, dtype="f16", table=False, lse=True,
             seen="all"),
        # A prompt's last 32 queries scoring a 65536-token INT2 cache (their log-sum-exps are not
        # known: no decode has run), each seeing the tokens up to its own.
        dict(name="weights_window", op="weights", queries=32, heads=32, kv_heads=8, dim=128,
             bits=2, group=32, block=128, tokens=65536, dtype="f16", table=True, lse=False,
             seen="causal"),
        # A ragged window: 17 queries, 12 query heads a KV head, 64-wide heads, a partly filled
        # last block, some queries that see nothing (padding).
        dict(name="weights_ragged", op="weights", queries=17, heads=24, kv_heads=2, dim=64, bits=4,
             group=32, block=128, tokens=10007, dtype="bf16", table=True, lse=False, seen="padded"),
        # A 131072-token cache halved, each KV head with its own choice.
        dict(name="evict_128k", op="evict", tokens=131072, keep=65536, kv_heads=8, dim=128, bits=4,
             group=32, block=128, sink=4, recent=4096, shared=False, table=False, mixed=False),
        # A small INT2 cache trimmed by a few blocks, one choice for all heads, after earlier
        # evictions have mixed the order of the tokens.
        dict(name="evict_shared", op="evict", tokens=10007, keep=8192, kv_heads=8, dim=128, bits=2,
             group=32, block=128, sink=4, recent=256, shared=True, table=True, mixed=True),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, evenly over the logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["rotary", "append", "weights", "evict"])
    dim = rng.choice([64, 96, 128, 128, 256])
    dtype = rng.choice(["f16", "bf16", "f32"])
    if op == "rotary":
        heads = rng.choice([1, 4, 8, 24, 32])
        return dict(op=op, tokens=_spread(rng, 1, 8192 * 4096 // (heads * dim * 2)), heads=heads,
                    dim=dim, part=rng.choice([dim, dim // 2]), dtype=dtype,
                    interleaved=rng.random() < 0.5,
                    scaling=rng.choice(["none", "linear", "smooth", "yarn"]),
                    far=_spread(rng, 16384, 1048576), strided=rng.random() < 0.5)
    kv_heads = rng.choice([1, 2, 4, 8])
    bits = rng.choice([2, 4])
    group = rng.choice([16, 32, dim // 2, dim])
    block = rng.choice([40, 64, 128])
    geometry = dict(kv_heads=kv_heads, dim=dim, bits=bits, group=group, block=block)
    if op == "append":
        tokens = _spread(rng, 1, 16384 * 1024 // (kv_heads * dim))
        return dict(op=op, tokens=tokens, **geometry, blocks=-(-tokens // block) + rng.randint(1, 40),
                    part=rng.choice([0, dim // 2, dim]), dtype=dtype,
                    interleaved=rng.random() < 0.5, far=_spread(rng, 131072, 1048576),
                    holes=rng.randint(0, min(3, tokens - 1)), outliers=rng.choice([0.0, 0.01]))
    tokens = _spread(rng, 100, 131072 * 1024 // (kv_heads * dim * 2))
    if op == "weights":
        per = rng.choice([1, 4, 8])
        most = max(1, 2**24 // (tokens * kv_heads * per))
        queries = rng.choice([1, _spread(rng, 1, min(64, most))])
        lse = queries == 1 and rng.random() < 0.7
        return dict(op=op, queries=queries, heads=per * kv_heads, **geometry, tokens=tokens,
                    dtype=dtype, table=rng.random() < 0.5, lse=lse,
                    seen="all" if lse else rng.choice(["all", "causal", "padded"]))
    sink, recent = rng.randint(0, 8), rng.randint(0, tokens // 8)
    return dict(op=op, tokens=tokens, keep=rng.randint(max(1, sink + recent), tokens - 1),
                **geometry, sink=sink, recent=recent, shared=rng.random() < 0.3,
                table=rng.random() < 0.5, mixed=rng.random() < 0.5)


def work(case):
    if case["op"] == "rotary":
        n = case["tokens"] * case["heads"] * case["dim"]
        return {"bytes": 2 * n * DTYPES[case["dtype"]].itemsize + 8 * case["tokens"],
                "flops": 3.0 * case["tokens"] * case["heads"] * case["part"]}
    rows = case["tokens"] * case["kv_heads"]
    row = case["dim"] * case["bits"] // 8 + 2 * (case["dim"] // case["group"])
    if case["op"] == "append":
        n = rows * case["dim"]
        return {"bytes": 2 * n * DTYPES[case["dtype"]].itemsize + 2 * rows * row + 2 * n * 2
                + 16 * case["tokens"], "flops": 2.0 * n * 4}
    if case["op"] == "weights":
        pairs = case["queries"] * case["heads"] * case["tokens"]
        return {"bytes": rows * row + 8 * rows
                + case["queries"] * case["heads"] * (case["dim"] * DTYPES[case["dtype"]].itemsize + 4),
                "flops": 2.0 * pairs * case["dim"]}
    # evict: weights read, weights and positions written over the cache's length, the kept ones'
    # positions read; the tokens kept from behind `keep` moved into the places before it
    moved = case["kv_heads"] * case["keep"] * (case["tokens"] - case["keep"]) / case["tokens"]
    return {"bytes": rows * 12 + case["kv_heads"] * case["keep"] * 4 + moved * 4 * row, "flops": 0.0}


# --------------------------------------------------------------------------------- inputs


def _frequencies(part, scaling, far):
    """Radians a position of each pair, in 64 bits: base 10000, stretched by 4 beyond a context of
    far / 4 in the way that `scaling` names. Returns (frequencies, magnitude of cos and sin)."""
    i = torch.arange(part // 2, dtype=torch.float64)
    freq = 10000.0 ** (-2.0 * i / part)
    if scaling == "none":
        return freq, 1.0
    factor, length = 4.0, far / 4.0
    if scaling == "linear":
        return freq / factor, 1.0
    turns = length * freq / (2 * math.pi)  # of each pair over the original context
    if scaling == "smooth":  # kept above 4 turns, divided below 1, in between by the turns
        keep = ((turns - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        return freq * keep + freq / factor * (1 - keep), 1.0
    # yarn: the ramp runs over the pair's index, between the pairs of 32 turns and of 1 turn
    at = [part * math.log(length / (b * 2 * math.pi)) / (2 * math.log(10000.0)) for b in (32.0, 1.0)]
    low, high = max(math.floor(at[0]), 0), min(math.ceil(at[1]), part - 1)
    ramp = ((i - low) / max(high - low, 1e-3)).clamp(0, 1)
    return freq / factor * ramp + freq * (1 - ramp), 0.1 * math.log(factor) + 1.0


def _quantize(x, bits, group):
    """Groupwise symmetric codes (0 .. 2^bits - 1) and FP16 scales of x (FP32) along its last axis;
    divisions by tensors, so that each is one correctly rounded FP32 division."""
    mid = 1 << (bits - 1)
    g = x.reshape(*x.shape[:-1], -1, group)
    scale = g.abs().amax(-1).clamp_min(1e-8) / torch.full((), float(mid - 1), device=x.device)
    codes = torch.round(g / scale.unsqueeze(-1)).clamp(-mid, mid - 1) + mid
    return codes.reshape(x.shape), scale.half()


def _pack(codes, bits):
    per = 8 // bits
    lanes = codes.to(torch.uint8).reshape(*codes.shape[:-1], -1, per)
    shifts = torch.arange(0, 8, bits, device=codes.device, dtype=torch.uint8)
    return (lanes << shifts).sum(-1).to(torch.uint8)


def _unpack(packed, bits):
    shifts = torch.arange(0, 8, bits, device=packed.device, dtype=torch.uint8)
    return ((packed.unsqueeze(-1) >> shifts) & ((1 << bits) - 1)).flatten(-2)


def _dequantize(packed, scales, bits):
    """(code - midpoint) * scale in FP32."""
    codes = _unpack(packed, bits).float() - (1 << (bits - 1))
    g = codes.reshape(*scales.shape, -1)
    return (g * scales.float().unsqueeze(-1)).reshape(codes.shape)


def _randn(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda")


def _table(gen, case, blocks):
    if not case["table"]:
        return None
    return torch.randperm(blocks, generator=gen, device="cuda").to(torch.int32)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    return {"case": case, **globals()["_prepare_" + case["op"]](case, gen)}


def _prepare_rotary(case, gen):
    t, h, d = case["tokens"], case["heads"], case["dim"]
    # strided: the leading heads of a wider projection (queries, keys and values in one row)
    x = _randn(gen, t, h + 2 if case["strided"] else h, d).to(DTYPES[case["dtype"]])[:, :h]
    start = torch.randint(0, max(1, case["far"] - t), (), generator=gen, device="cuda")
    freq, magnitude = _frequencies(case["part"], case["scaling"], case["far"])
    return {"x": x, "positions": torch.arange(t, device="cuda") + start, "frequencies": freq.cuda(),
            "magnitude": magnitude}


def _prepare_append(case, gen):
    t, h, d, bits = case["tokens"], case["kv_heads"], case["dim"], case["bits"]
    nb, bt = case["blocks"], case["block"]
    loud = torch.where(torch.rand(2, h, d, generator=gen, device="cuda") < case["outliers"], 8.0, 1.0)
    key, value = [(_randn(gen, t, h, d) * loud[i]).to(DTYPES[case["dtype"]]) for i in range(2)]
    slots = torch.randperm(nb * bt, generator=gen, device="cuda")[:t]  # a step: anywhere
    if t > 64:  # a prompt: in order through blocks in any order
        order = torch.randperm(nb, generator=gen, device="cuda")
        place = torch.arange(t, device="cuda") + torch.randint(0, bt, (), generator=gen, device="cuda")
        place = place.clamp_max(nb * bt - 1) if nb * bt >= t + bt else torch.arange(t, device="cuda")
        slots = order[place // bt] * bt + place % bt
    slots = slots.to(torch.int32)
    if case["holes"]:  # padding of the batch
        slots[torch.randperm(t, generator=gen, device="cuda")[:case["holes"]]] = -1
    start = torch.randint(0, max(1, case["far"] - t), (), generator=gen, device="cuda")
    freq = _frequencies(case["part"], "smooth", case["far"])[0].cuda() if case["part"] else None
    return {"key": key, "value": value, "slots": slots, "frequencies": freq,
            "positions": torch.arange(t, device="cuda") + start,
            "packed_k": torch.zeros(nb, bt, h, d * bits // 8, dtype=torch.uint8, device="cuda"),
            "packed_v": torch.zeros(nb, bt, h, d * bits // 8, dtype=torch.uint8, device="cuda"),
            "scales_k": torch.zeros(nb, bt, h, d // case["group"], dtype=torch.float16, device="cuda"),
            "scales_v": torch.zeros(nb, bt, h, d // case["group"], dtype=torch.float16, device="cuda"),
            "valid_tokens": torch.zeros(nb, dtype=torch.int32, device="cuda")}


def _prepare_weights(case, gen):
    tq, qh, h, d = case["queries"], case["heads"], case["kv_heads"], case["dim"]
    n, bt = case["tokens"], case["block"]
    nb = -(-n // bt)
    keys = _randn(gen, nb * bt, h, d)
    query = _randn(gen, tq, qh, d)
    # some tokens that many queries look at, as real contexts have them
    heavy = torch.rand(nb * bt, h, 1, generator=gen, device="cuda") < 0.01
    mean = query.reshape(tq, h, qh // h, d).mean((0, 2))
    keys = keys + heavy * 3.0 * mean / mean.norm(dim=-1, keepdim=True)
    codes, scales = _quantize(keys, case["bits"], case["group"])
    table = _table(gen, case, nb)
    valid = torch.full((nb,), bt, dtype=torch.int32, device="cuda")
    valid[nb - 1 if table is None else table[nb - 1]] = n - (nb - 1) * bt
    visible = None
    if case["seen"] != "all":
        visible = (n - tq + 1 + torch.arange(tq, device="cuda")).clamp_min(0).to(torch.int32)
        if case["seen"] == "padded":
            visible[tq // 2:tq // 2 + max(1, tq // 8)] = 0
    s = {"query": query.to(DTYPES[case["dtype"]]), "packed_k": _pack(codes, case["bits"]).reshape(nb, bt, h, -1),
         "scales_k": scales.reshape(nb, bt, h, -1), "valid_tokens": valid, "table": table,
         "visible": visible, "lse": None,
         "previous": torch.rand(h, nb * bt, generator=gen, device="cuda") * 0.01,
         "sm_scale": 1.0 / math.sqrt(d)}
    if case["lse"]:  # what the step's attention has returned beside its output
        scores = _scores({"case": case, **s})
        s["lse"] = torch.logsumexp(scores.double(), -1).float().transpose(0, 1).reshape(tq, qh)
    return s


def _prepare_evict(case, gen):
    n, h, bt, d = case["tokens"], case["kv_heads"], case["block"], case["dim"]
    nb = -(-n // bt)
    # heavy-tailed sums, a good part of them zero: ties that the lowest place decides
    weights = torch.exp(2.0 * _randn(gen, h, nb * bt))
    weights = weights * (torch.rand(h, nb * bt, generator=gen, device="cuda") > 0.2)
    if case["mixed"]:
        order = torch.rand(h, n, generator=gen, device="cuda").argsort(-1)
    else:
        order = torch.arange(n, device="cuda").expand(h, n)
    positions = torch.full((h, nb * bt), -1, dtype=torch.int32, device="cuda")
    positions[:, :n] = order
    if case["shared"]:  # one choice for all heads has left the same tokens in the same places
        positions = positions[:1].expand(h, -1).contiguous()
    table = _table(gen, case, nb)
    valid = torch.full((nb,), bt, dtype=torch.int32, device="cuda")
    valid[nb - 1 if table is None else table[nb - 1]] = n - (nb - 1) * bt
    pd, g = d * case["bits"] // 8, d // case["group"]
    codes = [torch.randint(0, 256, (nb, bt, h, pd), generator=gen, device="cuda", dtype=torch.uint8)
             for _ in range(2)]
    scales = [torch.rand(nb, bt, h, g, generator=gen, device="cuda").half() for _ in range(2)]
    return {"weights": weights, "positions": positions, "table": table, "valid_tokens": valid,
            "packed_k": codes[0], "packed_v": codes[1], "scales_k": scales[0], "scales_v": scales[1]}


# ------------------------------------------------------------------------------ plain forms


def _rotate(x, positions, frequencies, interleaved, magnitude):
    """x [tokens, heads, dim] in FP32 or FP64, its first 2 * len(frequencies) dims rotated; the angles
    in 64 bits (those of far positions lose too much in 32)."""
    part = 2 * frequencies.numel()
    angle = positions.double().unsqueeze(-1) * frequencies
    cos = (angle.cos() * magnitude).to(x.dtype).unsqueeze(1)
    sin = (angle.sin() * magnitude).to(x.dtype).unsqueeze(1)
    head, rest = x[..., :part], x[..., part:]
    if interleaved:
        a, b = head[..., 0::2], head[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = head[..., :part // 2], head[..., part // 2:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, rest], -1)


def _plain_rotary(s):
    c = s["case"]
    return _rotate(s["x"].float(), s["positions"], s["frequencies"], c["interleaved"],
                   s["magnitude"]).to(s["x"].dtype)


def _plain_append(s):
    c = s["case"]
    bits, group, bt = c["bits"], c["group"], c["block"]
    key = s["key"].float()
    if s["frequencies"] is not None:  # in 64 bits: codes lie on either side of a border
        key = _rotate(s["key"].double(), s["positions"], s["frequencies"], c["interleaved"], 1.0).float()
    live = s["slots"] >= 0
    to = s["slots"][live].long()
    values = []
    for x, packed, scales in ((key, s["packed_k"], s["scales_k"]),
                              (s["value"].float(), s["packed_v"], s["scales_v"])):
        codes, sc = _quantize(x, bits, group)
        packed.flatten(0, 1)[to] = _pack(codes, bits)[live]
        scales.flatten(0, 1)[to] = sc[live]
        centred = (codes - (1 << (bits - 1))).reshape(*sc.shape, group)
        values.append((centred * sc.float().unsqueeze(-1)).reshape(x.shape).half())
    s["valid_tokens"].scatter_reduce_(0, to // bt, (to % bt + 1).to(torch.int32), "amax")
    return values


def _scores(s):
    """Scaled scores [kv_heads, queries, heads a KV head, tokens] in FP32, -inf where masked."""
    c = s["case"]
    tq, h, bt = c["queries"], c["kv_heads"], c["block"]
    packed, scales, valid = s["packed_k"], s["scales_k"], s["valid_tokens"]
    if s["table"] is not None:
        at = s["table"].long()
        packed, scales, valid = packed[at], scales[at], valid[at]
    keys = _dequantize(packed, scales, c["bits"]).flatten(0, 1)
    query = s["query"].float().reshape(tq, h, -1, c["dim"])
    scores = torch.einsum("thgd,nhd->htgn", query, keys) * s["sm_scale"]
    place = torch.arange(keys.shape[0], device=keys.device)
    seen = (place % bt < valid.repeat_interleave(bt)).expand(tq, -1)
    if s["visible"] is not None:
        seen = seen & (place < s["visible"].unsqueeze(-1))
    return scores.masked_fill_(~seen[:, None], -math.inf)


def _plain_weights(s):
    c = s["case"]
    scores = _scores(s)
    if s["lse"] is None:
        top = scores.amax(-1, keepdim=True)
        top = torch.where(top == -math.inf, 0.0, top)
        lse = (scores - top).exp_().sum(-1).log() + top.squeeze(-1)
    else:
        lse = s["lse"].reshape(c["queries"], c["kv_heads"], -1).transpose(0, 1)
    empty = lse == -math.inf
    p = (scores - torch.where(empty, 0.0, lse).unsqueeze(-1)).exp_()
    return s["previous"] + p.sum((1, 2)), lse.transpose(0, 1).reshape(c["queries"], c["heads"])


def _plain_evict(s):
    c = s["case"]
    n, keep, h, bt = c["tokens"], c["keep"], c["kv_heads"], c["block"]
    w, pos = s["weights"][:, :n], s["positions"][:, :n]
    rank = w.double().sum(0, keepdim=True).float().expand(h, n) if c["shared"] else w
    safe = (pos < c["sink"]) | (pos >= n - c["recent"])
    rank = torch.where(safe, math.inf, rank)
    chosen = torch.sort(rank, dim=-1, descending=True, stable=True).indices[:, :keep]
    kept = torch.zeros(h, n, dtype=torch.bool, device=w.device).scatter_(1, chosen, True)
    # the i-th place to fill before `keep` takes the i-th kept token behind it
    late = kept[:, keep:]
    to = torch.where(late, late.cumsum(-1) - 1, n - keep)
    place = torch.arange(keep, n, device=w.device).expand(h, -1)
    movers = place.new_zeros(h, n - keep + 1).scatter_(1, to, place)
    holes = ~kept[:, :keep]
    source = torch.where(holes, movers.gather(1, (holes.cumsum(-1) - 1).clamp_min(0).clamp_max(n - keep)),
                         torch.arange(keep, device=w.device))
    weights = torch.zeros_like(s["weights"])
    weights[:, :keep] = w.gather(1, source)
    positions = torch.full_like(s["positions"], -1)
    positions[:, :keep] = pos.gather(1, source)
    nb = -(-n // bt)
    table = torch.arange(nb, device=w.device) if s["table"] is None else s["table"].long()
    at = lambda i: table[i // bt] * bt + i % bt  # noqa: E731
    head = torch.arange(h, device=w.device).unsqueeze(-1)
    rows, dest = at(source), at(torch.arange(keep, device=w.device)).expand(h, -1)
    for name in ("packed_k", "packed_v", "scales_k", "scales_v"):
        flat = s[name].flatten(0, 1)
        flat[dest, head] = flat[rows, head]
    left = (keep - bt * torch.arange(nb, device=w.device)).clamp(0, bt).to(torch.int32)
    s["valid_tokens"][table] = left
    return weights, positions


# -------------------------------------------------------------------------------------- run

_ops = None


def _framework():
    global _ops
    if _ops is None:
        package = str(Path("kvssd-attention_b200").resolve())
        if package not in sys.path:
            sys.path.insert(0, package)
        from kvssd_b200 import ops
        _ops = ops
    return _ops


def run(state):
    s, c = state, state["case"]
    op = c["op"]
    if own:
        ops = _ops or _framework()
        if op == "rotary":
            return ops.rotary(s["x"], s["positions"], s["frequencies"], interleaved=c["interleaved"],
                              magnitude=s["magnitude"])
        if op == "append":
            values = ops.append(s["key"], s["value"], s["slots"], s["packed_k"], s["packed_v"],
                                s["scales_k"], s["scales_v"], c["bits"], c["group"],
                                positions=s["positions"], frequencies=s["frequencies"],
                                interleaved=c["interleaved"], valid_tokens=s["valid_tokens"],
                                values=True)
        elif op == "weights":
            weights, lse = ops.attention_weights(
                s["query"], s["packed_k"], s["scales_k"], s["valid_tokens"], c["bits"], c["group"],
                s["sm_scale"], lse=s["lse"], block_table=s["table"], visible=s["visible"],
                previous=s["previous"])
        else:
            weights, positions = ops.evict(
                s["weights"], s["positions"], c["tokens"], c["keep"], s["packed_k"], s["packed_v"],
                s["scales_k"], s["scales_v"], s["valid_tokens"], block_table=s["table"],
                sink=c["sink"], recent=c["recent"], shared=c["shared"])
    elif op == "rotary":
        return _plain_rotary(s)
    elif op == "append":
        values = _plain_append(s)
    elif op == "weights":
        weights, lse = _plain_weights(s)
    else:
        weights, positions = _plain_evict(s)
    if op == "weights":
        return {"weights": weights, "lse": lse}
    # The pool's bytes and scales are the operators' result as well. The layout is shared with
    # stored records and fixed to the bit, so the bytes are returned as they are: they have to be
    # equal, not only stand for values that are near. `values` are what append's codes stand for.
    pool = {k: s[k] for k in ("packed_k", "packed_v", "scales_k", "scales_v", "valid_tokens")}
    if op == "append":
        return {"key": values[0], "value": values[1], **pool}
    return {"weights": weights, "positions": positions, **pool}


# ------------------------------------------------------------------------------------ exact


def _turned(x, s, c, magnitude):
    """The rotation as a product of complex numbers, in 64 bits."""
    x = x.double()
    part = 2 * s["frequencies"].numel()
    angle = torch.outer(s["positions"].double(), s["frequencies"])
    unit = torch.polar(torch.full_like(angle, magnitude), angle).unsqueeze(1)
    z = x[..., :part]
    if c["interleaved"]:
        z = torch.complex(z[..., 0::2].contiguous(), z[..., 1::2].contiguous()) * unit
        x[..., 0:part:2], x[..., 1:part:2] = z.real, z.imag
    else:
        z = torch.complex(z[..., :part // 2].contiguous(), z[..., part // 2:].contiguous()) * unit
        x[..., :part // 2], x[..., part // 2:part] = z.real, z.imag
    return x


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "rotary":
        return _turned(s["x"], s, c, s["magnitude"])
    if c["op"] == "append":
        mid, g = 1 << (c["bits"] - 1), c["group"]
        out = {"valid_tokens": None, "packed_k": None, "packed_v": None}
        key = s["key"].double() if s["frequencies"] is None else _turned(s["key"], s, c, 1.0)
        for name, x in (("key", key), ("value", s["value"].double())):
            groups = x.unflatten(-1, (-1, g))
            # the format's quantizer rounds the step and the quotient to FP32 (16-bit inputs hit
            # the border between two codes exactly, so these roundings belong to the definition)
            step = torch.maximum(groups.amax(-1), -groups.amin(-1)).float().double().clamp_min(1e-8)
            step = torch.true_divide(step, torch.full_like(step, mid - 1.0)).float().double()
            level = torch.round((groups.float().double() / step[..., None]).float().double())
            level = torch.clamp(level, -mid, mid - 1)
            held = step.half().double()  # scales are FP16 by the cache's format
            out[name] = (level * held[..., None]).flatten(-2)
            pool = torch.zeros(s["scales_" + name[0]].shape, dtype=torch.float64, device=x.device)
            rows = pool.view(-1, *pool.shape[2:])
            live = s["slots"] >= 0
            rows[s["slots"][live].long()] = held[live]
            out["scales_" + name[0]] = pool
        return out
    if c["op"] == "weights":
        tq, h, d = c["queries"], c["kv_heads"], c["dim"]
        nb, bt = s["packed_k"].shape[:2]
        blocks = torch.arange(nb, device="cuda") if s["table"] is None else s["table"].long()
        per = 8 // c["bits"]
        raw = s["packed_k"][blocks].long()
        codes = torch.stack([(raw // 2 ** (c["bits"] * i)) % 2 ** c["bits"] for i in range(per)], -1)
        keys = (codes.flatten(-2) - 2 ** (c["bits"] - 1)).double()
        keys = keys * s["scales_k"][blocks].double().repeat_interleave(c["group"], -1)
        keys = keys.reshape(nb * bt, h, d).permute(1, 2, 0)
        q = s["query"].double().reshape(tq, h, -1, d).permute(1, 0, 2, 3).reshape(h, -1, d)
        score = torch.bmm(q, keys).reshape(h, tq, -1, nb * bt) * s["sm_scale"]
        hidden = torch.arange(bt, device="cuda") >= s["valid_tokens"][blocks, None]
        score[..., hidden.flatten()] = -math.inf
        if s["visible"] is not None:
            later = torch.arange(nb * bt, device="cuda") >= s["visible"][:, None]
            score.masked_fill_(later[None, :, None], -math.inf)
        lse = torch.logsumexp(score, -1) if s["lse"] is None else s["lse"].double().reshape(
            tq, h, -1).transpose(0, 1)
        if s["lse"] is not None:
            p = torch.exp(score - lse[..., None])
        else:
            p = torch.softmax(score, -1).nan_to_num(0.0)  # a query that sees nothing gives nothing
        return {"weights": s["previous"].double() + p.sum((1, 2)),
                "lse": lse.transpose(0, 1).reshape(tq, -1)}
    # evict: the numbers are moved, not computed; the k-th largest by selection instead of sorting
    n, keep = c["tokens"], c["keep"]
    w = s["weights"][:, :n].double()
    if c["shared"]:
        w = w.sum(0, keepdim=True).float().double().expand_as(w)
    position = s["positions"][:, :n]
    w = w.masked_fill((position < c["sink"]) | (position >= n - c["recent"]), math.inf)
    new = torch.zeros_like(s["weights"], dtype=torch.float64)
    for head in range(c["kv_heads"]):
        border = torch.kthvalue(w[head], n - keep + 1).values
        above = torch.nonzero(w[head] > border).flatten()
        level = torch.nonzero(w[head] == border).flatten()[:keep - above.numel()]
        kept = torch.cat([above, level]).sort().values
        early, late = kept[kept < keep], kept[kept >= keep]
        new[head, early] = s["weights"][head, early].double()
        free = torch.ones(keep, dtype=torch.bool, device="cuda")
        free[early] = False
        new[head, torch.nonzero(free).flatten()] = s["weights"][head, late].double()
    return {"weights": new, "positions": None, "packed_k": None, "packed_v": None,
            "scales_k": None, "scales_v": None, "valid_tokens": None}
