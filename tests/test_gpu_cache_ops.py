"""Cache-maintenance operators on a B200 against their 64-bit restatement (oracle/cache_oracle.py).

Tolerances. A rounding to type t is off by at most eps_t / 2 of the value. rotary: FP32 cos and sin
of an angle reduced in FP64 and rounded to a fraction of a turn (2^-25 of a half turn, pi 2^-25 <
2^-23 rad; the functions themselves to 2 ulp, 2^-22) and two products and a sum (3 x 2^-24) leave
2^-21 (|a| + |b|) m, then one rounding to the type. append: codes, scales and values are exact.
attention_weights: a score is an FP32 sum of D exact products with at most 2^-22 on each operand, so
off by (D + 16) 2^-24 sum|q||k|, as is the log-sum-exp; a weight is off by twice that plus 2^-18
relative for the exponentials and the sum over up to 2^10 rows. evict moves and selects: exact."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from kvssd_b200 import CacheSpec, DeviceBlockPool, DeviceKVCache, RotaryEmbedding, _native, ops
from kvssd_b200.quant import dequantize_tensor, quantize_tensor
from oracle import cache_oracle as orc

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = {"f32": 2.0**-23, "f16": 2.0**-10, "bf16": 2.0**-7}


def gen(seed):
    return torch.Generator().manual_seed(seed)


def freqs(pairs, base=10000.0):
    return base ** (-torch.arange(pairs, dtype=torch.float64) / pairs)


# ------------------------------------------------------------------------------------ rotary


def check_rotary(x, positions, f, interleaved, magnitude, out, name):
    ref = orc.rotate(x.double().cpu().numpy(), positions.cpu().numpy(), f.numpy(), interleaved, magnitude)
    mag = orc.rotate(x.double().abs().cpu().numpy(), np.zeros(len(positions)), f.numpy(), interleaved)
    half = 2 * len(f)
    both = np.abs(mag).copy()
    rot = both[..., :half]
    pair = (rot.reshape(*rot.shape[:-1], -1, 2).sum(-1).repeat(2, -1) if interleaved else
            np.concatenate([rot[..., :half // 2] + rot[..., half // 2:]] * 2, -1))
    tol = np.zeros_like(ref)
    tol[..., :half] = pair * magnitude * 2.0**-21
    tol += np.abs(ref) * EPS[name] / 2 + 2.0**-25  # FP16 subnormals: half of 2^-24
    got = out.double().cpu().numpy()
    assert (np.abs(got - ref) <= tol).all(), np.max(np.abs(got - ref) - tol)
    np.testing.assert_array_equal(got[..., half:], x.double().cpu().numpy()[..., half:])


@pytest.mark.parametrize("name", list(TYPES))
@pytest.mark.parametrize("tokens, heads, d, pairs", [
    (1, 1, 64, 32), (1, 32, 128, 64), (3, 24, 64, 16), (7, 5, 96, 48), (129, 8, 128, 32),
    (1000, 2, 256, 128), (5, 3, 20, 7), (33, 130, 128, 64), (2, 1, 2, 1), (300, 1, 128, 64)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary(tokens, heads, d, pairs, interleaved, name):
    x = torch.randn(tokens, heads, d, generator=gen(tokens + d)).to(TYPES[name]).to(DEV)
    positions = torch.arange(tokens, device=DEV) * 997 + 1_000_003
    if tokens > 2:
        positions[1], positions[2] = 0, -5
    f = freqs(pairs)
    out = ops.rotary(x, positions, f.to(DEV), interleaved=interleaved, magnitude=1.25)
    check_rotary(x, positions, f, interleaved, 1.25, out, name)


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_strided_in_place_and_int32(interleaved):
    f = freqs(24)
    wide = torch.randn(37, 12, 64, generator=gen(1)).half().to(DEV)
    before = wide.clone()
    positions = torch.arange(37, device=DEV, dtype=torch.int32) + 77
    ref = ops.rotary(before[:, 3:8].contiguous(), positions.long(), f.to(DEV), interleaved=interleaved)
    part = wide[:, 3:8]
    assert ops.rotary(part, positions, f.to(DEV), interleaved=interleaved, out=part) is part
    assert torch.equal(part, ref)
    assert torch.equal(wide[:, :3], before[:, :3]) and torch.equal(wide[:, 8:], before[:, 8:])
    # heads-first storage, odd token stride, an expanded input, an unaligned start
    first = before[:, 3:8].transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(ops.rotary(first, positions, f.to(DEV), interleaved=interleaved), ref)
    odd = torch.empty(37 * (5 * 64 + 1) + 3, dtype=torch.float16, device=DEV)
    view = odd[3:].as_strided((37, 5, 64), (5 * 64 + 1, 64, 1))
    view.copy_(before[:, 3:8])
    assert torch.equal(ops.rotary(view, positions, f.to(DEV), interleaved=interleaved), ref)
    one = before[:1, 3:8].expand(37, 5, 64)
    again = ops.rotary(one.contiguous(), positions, f.to(DEV), interleaved=interleaved)
    assert torch.equal(ops.rotary(one, positions, f.to(DEV), interleaved=interleaved), again)
    last = before[:, 3:8].transpose(1, 2).contiguous().transpose(1, 2)  # last dim strided: copied
    assert torch.equal(ops.rotary(last, positions, f.to(DEV), interleaved=interleaved), ref)


def test_rotary_empty_and_refusals():
    f = freqs(4).to(DEV)
    x = torch.randn(2, 3, 8, device=DEV)
    pos = torch.arange(2, device=DEV)
    assert ops.rotary(x[:0], pos[:0], f).shape == (0, 3, 8)
    for bad in (lambda: ops.rotary(x.double(), pos, f), lambda: ops.rotary(x[0], pos, f),
                lambda: ops.rotary(x, pos[:1], f), lambda: ops.rotary(x, pos.float(), f),
                lambda: ops.rotary(x, pos.cpu(), f), lambda: ops.rotary(x, pos, f.float()),
                lambda: ops.rotary(x, pos, f.cpu()), lambda: ops.rotary(x, pos, freqs(5).to(DEV)),
                lambda: ops.rotary(x, pos, f[:0]), lambda: ops.rotary(x, pos, f, out=x.half()),
                lambda: ops.rotary(x, pos, f, out=torch.empty(1, 3, 8, device=DEV).expand(2, 3, 8))):
        with pytest.raises(ValueError):
            bad()


def test_rotary_embedding_applies_its_scaling():
    emb = RotaryEmbedding(64, rotary_dim=32, interleaved=True, scaling="yarn", factor=4.0,
                          original_length=4096)
    x = torch.randn(9, 2, 64, generator=gen(3)).to(DEV)
    pos = torch.arange(9, device=DEV) + 10_000
    out = emb.apply(x, pos)
    check_rotary(x, pos, emb.frequencies(), True, emb.magnitude, out, "f32")
    assert emb.on("cuda") is emb.on(DEV)


# ------------------------------------------------------------------------------------ append


def make_pool(nb, bt, kvh, d, bits, group, fill=0):
    codes = [torch.full((nb, bt, kvh, d * bits // 8), fill, dtype=torch.uint8, device=DEV) for _ in "kv"]
    scales = [torch.full((nb, bt, kvh, d // group), float(fill), dtype=torch.float16, device=DEV)
              for _ in "kv"]
    return [*codes, *scales]


def quantized(x32, bits, group):
    q = quantize_tensor(x32, bits, group)  # on the CPU: the reference's bits
    return q.packed, q.scales, dequantize_tensor(q, torch.float16)


CASES = [  # tokens, kvh, d, bits, group, bt, pairs
    (1, 8, 128, 4, 32, 128, 64), (16, 8, 128, 4, 32, 128, 0), (100, 2, 64, 2, 16, 40, 32),
    (37, 1, 96, 4, 48, 8, 24), (5, 3, 128, 2, 64, 16, 64), (300, 8, 128, 2, 32, 128, 32),
    (9, 2, 256, 4, 256, 12, 128), (12, 1, 36, 4, 12, 8, 5), (64, 4, 256, 4, 128, 64, 64),
    (7, 5, 64, 4, 64, 8, 32), (1, 1, 8, 2, 4, 4, 4), (40, 1, 128, 4, 8, 16, 0), (33, 2, 96, 2, 96, 8, 48)]


@pytest.mark.parametrize("name", list(TYPES))
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("case", CASES)
def test_append(case, interleaved, name):
    tokens, kvh, d, bits, group, bt, pairs = case
    g = gen(sum(case))
    key, value = [(torch.randn(tokens, kvh, d, generator=g) * 2).to(TYPES[name]) for _ in "kv"]
    nb = -(-tokens // bt) + 2
    slots = torch.randperm(nb * bt, generator=g)[:tokens]
    slots[tokens // 2] = -1
    positions = torch.arange(tokens) * 13 + 123_457
    pool = make_pool(nb, bt, kvh, d, bits, group, fill=3)
    expect = [t.cpu().clone() for t in pool]
    valid = torch.zeros(nb, dtype=torch.int32, device=DEV)
    valid[0] = bt
    turn = {}
    k32 = key.float()
    if pairs:
        f = freqs(pairs)
        turn = dict(positions=positions.to(DEV), frequencies=f.to(DEV), interleaved=interleaved,
                    magnitude=1.0)
        k32 = torch.from_numpy(orc.rotate(key.double().numpy(), positions.numpy(), f.numpy(),
                                          interleaved).astype(np.float32))
    held = ops.append(key.to(DEV), value.to(DEV), slots.to(DEV), *pool, bits, group,
                      valid_tokens=valid, values=True, **turn)
    live = slots >= 0
    for i, x in enumerate((k32, value.float())):
        packed, scales, values = quantized(x, bits, group)
        expect[i].flatten(0, 1)[slots[live]] = packed[live]
        expect[2 + i].flatten(0, 1)[slots[live]] = scales[live]
        assert torch.equal(held[i].cpu(), values)
    for got, ref in zip(pool, expect):
        assert torch.equal(got.cpu(), ref)
    counts = torch.zeros(nb, dtype=torch.int32)
    counts[0] = bt
    for s in slots[live].tolist():
        counts[s // bt] = max(counts[s // bt], s % bt + 1)
    assert torch.equal(valid.cpu(), counts)
    assert ops.read_device_status(DEV) == 0


MANY = [  # so many tokens that a warp takes several of them, or two or four steps of heads
    (2049, 1, 64, 4, 32, 40, 32), (1501, 1, 128, 2, 64, 64, 32), (1203, 2, 128, 4, 16, 128, 64),
    (1301, 3, 96, 4, 32, 24, 48), (1999, 1, 16, 2, 8, 24, 8), (1250, 5, 40, 4, 8, 16, 16), (1250, 2, 24, 2, 24, 16, 8),
    (1301, 4, 128, 2, 32, 64, 64), (1190, 2, 256, 4, 64, 32, 64), (1187, 7, 128, 4, 32, 64, 64), (2500, 1, 8, 4, 8, 64, 0)]


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("case", MANY)
def test_append_many_tokens(case, interleaved, name):
    test_append(case, interleaved, name)


def test_append_strided_int32_and_without_values():
    pool, again = (make_pool(4, 16, 4, 128, 4, 32) for _ in range(2))
    g = gen(8)
    qkv = torch.randn(20, 12, 128, generator=g).bfloat16().to(DEV)
    slots = torch.randperm(64, generator=g)[:20].to(DEV)
    pos = torch.arange(20, device=DEV)
    f = freqs(64).to(DEV)
    assert ops.append(qkv[:, 4:8], qkv[:, 8:], slots, *pool, 4, 32, positions=pos, frequencies=f) is None
    ops.append(qkv[:, 4:8].contiguous(), qkv[:, 8:].contiguous(), slots.int(), *again, 4, 32,
               positions=pos.int(), frequencies=f)
    assert all(torch.equal(a, b) for a, b in zip(pool, again))
    odd = torch.empty(20 * 1537 + 1, dtype=torch.bfloat16, device=DEV)  # no 16-byte alignment
    view = odd[1:].as_strided((20, 12, 128), (1537, 128, 1))
    view.copy_(qkv)
    third = make_pool(4, 16, 4, 128, 4, 32)
    ops.append(view[:, 4:8], view[:, 8:], slots, *third, 4, 32, positions=pos, frequencies=f)
    assert all(torch.equal(a, b) for a, b in zip(pool, third))


@pytest.mark.parametrize("d, group", [(128, 32), (20, 4)])
def test_append_odd_values(d, group):
    """Zeros, ties between two codes, tiny and huge groups, infinities and a NaN: groups of finite
    values equal the quantizer's, a NaN or an infinity shows in its own group's scale only."""
    x = torch.randn(6, 1, d, generator=gen(2))
    x[0] = 0.0
    x[1, 0] = torch.arange(d) % 15 - 7.0  # quotients that are whole
    x[1, 0, 0::2] += 0.5  # and halves: ties
    x[1, 0, :: group] = 7.0
    x[2] *= 1e-12
    x[3] *= 1e6  # scales beyond FP16: infinite, as the quantizer's
    y = x.clone()
    y[4, 0, 1], y[5, 0, group + 1] = math.inf, math.nan
    pool = make_pool(1, 8, 1, d, 4, group)
    slots = torch.arange(6, device=DEV)
    ops.append(y.to(DEV), x.to(DEV), slots, *pool, 4, group)
    packed, scales, _ = quantized(x, 4, group)
    assert torch.equal(pool[1][0, :6].cpu(), packed) and torch.equal(pool[3][0, :6].cpu(), scales)
    k, s = pool[0][0, :6].cpu(), pool[2][0, :6].cpu()
    assert math.isinf(s[4, 0, 0]) and math.isnan(s[5, 0, 1])
    s[4, 0, 0], s[5, 0, 1] = scales[4, 0, 0], scales[5, 0, 1]
    assert torch.equal(s, scales)
    b = group // 2
    k[4, 0, :b], k[5, 0, b:2 * b] = packed[4, 0, :b], packed[5, 0, b:2 * b]
    assert torch.equal(k, packed)


def test_append_refuses_slots_behind_the_pool():
    ops.read_device_status(DEV)
    pool = make_pool(2, 4, 1, 32, 4, 16)
    x = torch.randn(3, 1, 32, device=DEV)
    slots = torch.tensor([8, 1, 2**40], device=DEV)
    ops.append(x, x, slots, *pool, 4, 16)
    assert ops.read_device_status(DEV) == _native.DEV_BAD_BLOCK
    rows = pool[2].flatten(0, 1)
    assert (rows[1] != 0).all() and (rows[[0, 2, 3, 4, 5, 6, 7]] == 0).all()


def test_append_refusals_and_empty():
    pool = make_pool(2, 4, 1, 32, 4, 16)
    x = torch.randn(3, 1, 32, device=DEV)
    s = torch.arange(3, device=DEV)
    f = freqs(16).to(DEV)
    assert ops.append(x[:0], x[:0], s[:0], *pool, 4, 16) is None
    for bad in (lambda: ops.append(x.double(), x.double(), s, *pool, 4, 16),
                lambda: ops.append(x, x.half(), s, *pool, 4, 16),
                lambda: ops.append(x, x[:2], s, *pool, 4, 16),
                lambda: ops.append(x, x, s.float(), *pool, 4, 16),
                lambda: ops.append(x, x, s, *pool, 2, 16), lambda: ops.append(x, x, s, *pool, 4, 8),
                lambda: ops.append(x, x, s, *pool, 4, 16, frequencies=f),
                lambda: ops.append(x, x, s, *pool, 4, 16, valid_tokens=s),
                lambda: ops.append(x, x, s, pool[0][:, ::2], pool[1], pool[2], pool[3], 4, 16),
                lambda: ops.append(x.transpose(1, 2).expand(3, 32, 32), x, s, *pool, 4, 16)):
        with pytest.raises(ValueError):
            bad()


# --------------------------------------------------------------------------- attention weights


def key_pool(nb, bt, kvh, d, bits, group, seed, outliers=False):
    k = torch.randn(nb, bt, kvh, d, generator=gen(seed)) * 1.5
    if outliers:
        k[..., :: 17] *= 8.0
    q = quantize_tensor(k, bits, group)
    return q.packed.to(DEV), q.scales.to(DEV)


def check_weights(query, kp, ks, valid, bits, group, scale, *, lse=None, table=None, visible=None,
                  previous=None, got=None, given=None):
    q3 = query.double().cpu().numpy().reshape(-1, *query.shape[-2:])
    cpu = lambda t: None if t is None else t.cpu().numpy()  # noqa: E731
    w, full, bound = orc.attention_weights(
        q3, cpu(kp), cpu(ks), cpu(valid), bits, group, scale, table=cpu(table), visible=cpu(visible),
        lse=None if lse is None else cpu(lse).reshape(q3.shape[:2]))
    off = (q3.shape[-1] + 16) * 2.0**-24 * bound  # of a score and of a log-sum-exp
    prev = 0.0 if previous is None else previous.double().cpu().numpy()
    tol = w * (np.expm1(2 * off) + 2.0**-18) + (np.abs(prev) + w) * 2.0**-23 + 1e-37
    out, out_lse = got
    mine = out.double().cpu().numpy()
    d = np.abs(mine - (w + prev))
    broken = np.isnan(w)  # an infinite scale times a zero code: the kernel says so too
    assert np.array_equal(np.isnan(mine), broken)
    assert (d <= tol)[~broken].all(), (d - tol)[~broken].max()
    if lse is None:
        l = out_lse.double().cpu().numpy().reshape(full.shape)
        assert np.array_equal(l == -np.inf, full == -np.inf)
        assert np.array_equal(np.isnan(l), np.isnan(full))
        live = np.isfinite(full)
        assert (np.abs(l - full)[live] <= off.max() + 2.0**-20 + 2.0**-23 * np.abs(full[live])).all()


W_CASES = [  # nb, bt, kvh, gqa, d, bits, group, queries
    (1, 1, 1, 1, 64, 4, 32, 1), (3, 128, 8, 4, 128, 4, 32, 1), (5, 40, 2, 12, 64, 4, 32, 3),
    (4, 128, 8, 4, 128, 2, 32, 2), (2, 128, 4, 8, 128, 4, 64, 5), (7, 16, 1, 8, 256, 4, 64, 1),
    (2, 24, 2, 4, 96, 4, 48, 2), (3, 8, 3, 1, 128, 4, 16, 4), (2, 128, 2, 1, 128, 4, 128, 17),
    (3, 64, 1, 3, 64, 2, 64, 9), (9, 10, 2, 5, 32, 2, 8, 1), (2, 32, 1, 16, 128, 2, 64, 40),
    (3, 37, 4, 2, 256, 2, 128, 2), (33, 16, 2, 7, 64, 2, 32, 11), (2, 16, 1, 4, 36, 4, 12, 3)]


@pytest.mark.parametrize("name", ["f32", "f16", "bf16", "f64"])
@pytest.mark.parametrize("case", W_CASES)
def test_weights(case, name):
    nb, bt, kvh, gqa, d, bits, group, queries = case
    g = gen(sum(case))
    kp, ks = key_pool(nb, bt, kvh, d, bits, group, 5, outliers=bits == 2)
    query = (torch.randn(queries, kvh * gqa, d, generator=g) * 1.3).to(
        {**TYPES, "f64": torch.float64}[name]).to(DEV)
    valid = torch.full((nb,), bt, dtype=torch.int32)
    valid[nb // 2] = bt // 3
    if nb > 2:
        valid[0] = 0
    valid = valid.to(DEV)
    table = torch.randint(0, nb, (nb + 2,), generator=g).int().to(DEV)
    previous = torch.rand(kvh, (nb + 2) * bt, generator=g).to(DEV)
    scale = 1 / math.sqrt(d)
    got = ops.attention_weights(query, kp, ks, valid, bits, group, scale)
    check_weights(query, kp, ks, valid, bits, group, scale, got=got)
    got = ops.attention_weights(query, kp, ks, valid, bits, group, scale, block_table=table,
                                previous=previous)
    check_weights(query, kp, ks, valid, bits, group, scale, table=table, previous=previous, got=got)
    lse = got[1] + 0.25  # given: whatever it is
    given = ops.attention_weights(query, kp, ks, valid, bits, group, scale, block_table=table, lse=lse)
    assert given[1] is lse
    check_weights(query, kp, ks, valid, bits, group, scale, table=table, lse=lse, got=given)


WINDOWS = [  # nb, bt, kvh, gqa, d, bits, group, queries
    (3, 128, 2, 4, 128, 4, 32, 32), (3, 128, 2, 4, 128, 2, 32, 32), (7, 40, 1, 12, 64, 4, 64, 5),
    (5, 100, 3, 1, 96, 4, 32, 50), (5, 100, 2, 2, 96, 2, 96, 33), (9, 64, 2, 8, 128, 4, 128, 40),
    (40, 17, 1, 3, 64, 2, 32, 64), (1, 1, 1, 33, 128, 4, 32, 1), (2, 300, 1, 129, 64, 4, 32, 2),
    (2, 128, 2, 4, 256, 4, 64, 40), (3, 70, 1, 4, 256, 2, 32, 63), (2, 128, 1, 4, 256, 2, 256, 10),
    (2, 100, 2, 4, 128, 4, 16, 30), (2, 100, 1, 5, 96, 2, 48, 11), (3, 30, 1, 40, 256, 4, 16, 1),
    (2, 64, 2, 40, 64, 2, 16, 1), (5, 8, 1, 50, 96, 4, 16, 3)]


@pytest.mark.parametrize("name", ["f32", "f16", "bf16", "f64"])
@pytest.mark.parametrize("case", WINDOWS)
def test_weights_windows(case, name):
    """More than 32 query rows a KV head: causal, padded, with given and computed log-sum-exps."""
    nb, bt, kvh, gqa, d, bits, group, queries = case
    g = gen(sum(case))
    kp, ks = key_pool(nb, bt, kvh, d, bits, group, 6, outliers=bits == 2)
    query = (torch.randn(queries, kvh * gqa, d, generator=g) * 1.3).to(
        {**TYPES, "f64": torch.float64}[name]).to(DEV)
    n = nb * bt - bt // 3
    valid = torch.full((nb,), bt, dtype=torch.int32)
    valid[-1] = bt - bt // 3
    valid = valid.to(DEV)
    visible = (n - queries + 1 + torch.arange(queries)).int()
    visible[queries // 2] = 0
    visible = visible.to(DEV)
    previous = torch.rand(kvh, nb * bt, generator=g).to(DEV)
    table = torch.randint(0, nb, (nb + 1,), generator=g).int().to(DEV)
    scale = 1 / math.sqrt(d)
    got = ops.attention_weights(query, kp, ks, valid, bits, group, scale)
    check_weights(query, kp, ks, valid, bits, group, scale, got=got)
    got = ops.attention_weights(query, kp, ks, valid, bits, group, -scale, visible=visible, previous=previous)
    check_weights(query, kp, ks, valid, bits, group, -scale, visible=visible, previous=previous, got=got)
    lse = got[1] + 0.25
    given = ops.attention_weights(query, kp, ks, valid, bits, group, scale, block_table=table, lse=lse)
    check_weights(query, kp, ks, valid, bits, group, scale, table=table, lse=lse, got=given)
    zero = ops.attention_weights(query, kp, ks, valid, bits, group, 0.0, visible=visible)
    check_weights(query, kp, ks, valid, bits, group, 0.0, visible=visible, got=zero)


SMALL_WINDOWS = [  # nb, bt, kvh, gqa, d, bits, group, queries: 9 to 32 rows, or shapes without tcgen05
    (3, 128, 2, 4, 128, 4, 32, 7), (3, 60, 1, 3, 128, 2, 32, 10), (4, 33, 2, 5, 64, 4, 64, 2),
    (4, 33, 3, 1, 64, 2, 32, 30), (3, 50, 2, 3, 96, 4, 96, 4), (3, 50, 2, 3, 96, 2, 48, 9),
    (2, 128, 1, 4, 256, 4, 64, 20), (3, 40, 2, 2, 256, 2, 256, 25), (2, 128, 2, 4, 128, 4, 16, 30),
    (2, 128, 2, 4, 64, 2, 16, 30), (2, 20, 1, 2, 256, 4, 16, 100), (3, 16, 1, 1, 128, 2, 16, 300)]


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("case", SMALL_WINDOWS)
def test_weights_small_windows(case, name):
    nb, bt, kvh, gqa, d, bits, group, queries = case
    g = gen(sum(case))
    kp, ks = key_pool(nb, bt, kvh, d, bits, group, 7, outliers=bits == 2)
    query = (torch.randn(queries, kvh * gqa, d, generator=g) * 1.3).to(TYPES[name]).to(DEV)
    valid = torch.full((nb,), bt, dtype=torch.int32, device=DEV)
    valid[-1] = bt // 2
    visible = (nb * bt - bt // 2 - queries + 1 + torch.arange(queries)).clamp_min(0).int().to(DEV)
    previous = torch.rand(kvh, nb * bt, generator=g).to(DEV)
    scale = 1 / math.sqrt(d)
    got = ops.attention_weights(query, kp, ks, valid, bits, group, scale, visible=visible, previous=previous)
    check_weights(query, kp, ks, valid, bits, group, scale, visible=visible, previous=previous, got=got)
    lse = got[1] - 0.25
    got = ops.attention_weights(query, kp, ks, valid, bits, group, scale, lse=lse)
    check_weights(query, kp, ks, valid, bits, group, scale, lse=lse, got=got)


def test_windows_in_graphs_and_on_two_streams():
    """The tensor-memory kernel beside itself: two captured windows replayed on two streams."""
    kp, ks = key_pool(12, 128, 4, 128, 4, 32, 2)
    valid = torch.full((12,), 128, dtype=torch.int32, device=DEV)
    queries = [torch.randn(40, 16, 128, generator=gen(i)).half().to(DEV) for i in range(2)]
    call = lambda q: ops.attention_weights(q, kp, ks, valid, 4, 32, 0.09)  # noqa: E731
    ref = [[t.clone() for t in call(q)] for q in queries]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(queries[0])
    torch.cuda.synchronize()
    graphs, outs = [], []
    for q in queries:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs.append(call(q))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(5):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
                graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(ref, outs):
            assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert ops.read_device_status_all(DEV) == 0


@pytest.mark.parametrize("bits", [2, 4])
@pytest.mark.parametrize("queries", [1, 16])
def test_weights_scales_at_the_end_of_fp16(bits, queries):
    """Key scales up to FP16's largest number (code times scale leaves FP16's range) and down to its
    smallest, in different tiles and beside each other; the scale brings the scores back to size. In
    FP16 the largest ones round to infinity: those keys' scores are not numbers, here and there."""
    kp, ks = key_pool(6, 128, 2, 128, bits, 32, 4)
    ks[0] *= 65504 / ks[0].max()
    ks[1, ::2] *= 30000 / ks[1].max()
    ks[2] = 2.0**-24
    ks[3, 5:9] = 6e-8
    valid = torch.full((6,), 128, dtype=torch.int32, device=DEV)
    query = torch.randn(queries, 8, 128, generator=gen(6)).to(DEV)
    for finite in (False, True):
        if finite:
            ks.clamp_(max=65504)
        for t, scale in ((torch.float32, 1e-6), (torch.float16, 2e-6)):
            got = ops.attention_weights(query.to(t), kp, ks, valid, bits, 32, scale)
            check_weights(query.to(t), kp, ks, valid, bits, 32, scale, got=got)


@pytest.mark.parametrize("geometry", [(4, 32, 8, 4, 128, 4, 32), (4, 20, 2, 3, 96, 4, 48),
                                      (3, 100, 2, 12, 128, 4, 32), (3, 100, 2, 12, 64, 2, 32)])
def test_weights_masks_and_odd_values(geometry):
    nb, bt, kvh, gqa, d, bits, group = geometry
    kp, ks = key_pool(nb, bt, kvh, d, bits, group, 9)
    valid = torch.full((nb,), bt, dtype=torch.int32, device=DEV)
    valid[-1] = 3
    ks[-1, 3:] = math.nan  # behind the valid rows
    kp[-1, 3:] = 255
    query = torch.randn(5, kvh * gqa, d, generator=gen(1)).half().to(DEV)
    n = nb * bt
    visible = torch.tensor([0, 1, n // 2 + 1, -7, 10**9], dtype=torch.int32, device=DEV)
    got = ops.attention_weights(query, kp, ks, valid, bits, group, 0.1, visible=visible)
    check_weights(query, kp, ks, valid, bits, group, 0.1, visible=visible, got=got)
    w, lse = got
    assert (w[:, (nb - 1) * bt + 3:] == 0).all()
    assert (lse[0] == -math.inf).all() and (lse[3] == -math.inf).all()
    # rows that see nothing, given as -inf; a NaN log-sum-exp shows in the places its query sees
    only = torch.full((5, kvh * gqa), -math.inf, device=DEV)
    assert (ops.attention_weights(query, kp, ks, valid, bits, group, 0.1, lse=only)[0] == 0).all()
    only[2] = math.nan
    w = ops.attention_weights(query, kp, ks, valid, bits, group, 0.1, lse=only, visible=visible)[0]
    assert w[:, :n // 2 + 1].isnan().all() and (w[:, n // 2 + 1:] == 0).all()
    none = torch.zeros_like(valid)
    w, lse = ops.attention_weights(query, kp, ks, none, bits, group, 0.1)
    assert (w == 0).all() and (lse == -math.inf).all()
    # scores far apart and far from zero
    got = ops.attention_weights(query * 30, kp, ks, valid, bits, group, 1.0)
    check_weights(query * 30, kp, ks, valid, bits, group, 1.0, got=got)
    got = ops.attention_weights(query, kp, ks, valid, bits, group, -0.5)
    check_weights(query, kp, ks, valid, bits, group, -0.5, got=got)
    zero = ops.attention_weights(query * 0, kp, ks, valid, bits, group, 0.1)
    check_weights(query * 0, kp, ks, valid, bits, group, 0.1, got=zero)


@pytest.mark.parametrize("geometry", [(2, 2, 128, 4, 32, 4), (6, 4, 128, 4, 32, 4), (12, 4, 64, 2, 32, 4),
                                      (6, 2, 32, 4, 8, 4), (12, 4, 256, 4, 64, 1), (2, 3, 96, 2, 16, 1)])
def test_weights_padding_queries_may_hold_anything(geometry):
    """Queries that see nothing, beside ones that see all, are NaN and infinite: nothing of them shows."""
    queries, gqa, d, bits, group, kvh = geometry
    kp, ks = key_pool(5, 64, kvh, d, bits, group, 12)
    valid = torch.full((5,), 64, dtype=torch.int32, device=DEV)
    clean = torch.randn(queries, kvh * gqa, d, generator=gen(2)).half().to(DEV)
    visible = torch.full((queries,), 10**6, dtype=torch.int32, device=DEV)
    visible[1::3], visible[2::3] = 0, -2**31
    padded = clean.clone()
    padded[1::3], padded[2::3] = math.nan, math.inf
    want = ops.attention_weights(clean, kp, ks, valid, bits, group, 0.1, visible=visible)
    check_weights(clean, kp, ks, valid, bits, group, 0.1, visible=visible, got=want)
    got = ops.attention_weights(padded, kp, ks, valid, bits, group, 0.1, visible=visible)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    for seen in (visible, None):  # None: the -inf log-sum-exps alone tell
        # the log-sum-exp goes through natural units: three roundings at its size, below 16
        w, _ = ops.attention_weights(padded, kp, ks, valid, bits, group, 0.1, visible=seen, lse=want[1])
        torch.testing.assert_close(w, want[0], rtol=1e-5, atol=0)


@pytest.mark.parametrize("scale", [1e-6, 1.0, 3e4])
def test_weights_query_ranges(scale):
    """FP32 and BF16 queries far outside FP16's range, with elements of very different size."""
    kp, ks = key_pool(3, 64, 2, 128, 4, 32, 4)
    valid = torch.full((3,), 64, dtype=torch.int32, device=DEV)
    query = torch.randn(3, 8, 128, generator=gen(6)) * 10.0 ** torch.linspace(-6, 0, 128)
    for t in (torch.float32, torch.bfloat16):
        q = (query * scale * 10).to(t).to(DEV)
        got = ops.attention_weights(q, kp, ks, valid, 4, 32, 0.1 / scale)
        check_weights(q, kp, ks, valid, 4, 32, 0.1 / scale, got=got)


def test_weights_in_place_views_and_single_query():
    kp, ks = key_pool(4, 128, 8, 128, 4, 32, 2)
    valid = torch.full((4,), 128, dtype=torch.int32, device=DEV)
    query = torch.randn(32, 128, generator=gen(3)).half().to(DEV)
    wide = torch.rand(8, 1000, generator=gen(4)).to(DEV)
    before = wide.clone()
    ref, lse = ops.attention_weights(query, kp, ks, valid, 4, 32, 0.09, previous=before[:, 100:612])
    assert lse.shape == (32,)
    view = wide[:, 100:612]
    out, _ = ops.attention_weights(query, kp, ks, valid, 4, 32, 0.09, previous=view, out=view)
    assert out is view and torch.equal(view, ref)
    assert torch.equal(wide[:, :100], before[:, :100]) and torch.equal(wide[:, 612:], before[:, 612:])
    # an odd start: no vector accesses
    odd = torch.empty(kp.numel() + 1, dtype=torch.uint8, device=DEV)[1:].view(kp.shape)
    odd.copy_(kp)
    got = ops.attention_weights(query, odd, ks, valid, 4, 32, 0.09)
    check_weights(query, kp, ks, valid, 4, 32, 0.09, got=got)


def test_weights_agree_with_decode():
    kp, ks = key_pool(20, 128, 8, 128, 4, 32, 2)
    vp, vs = key_pool(20, 128, 8, 128, 4, 32, 3)
    valid = torch.full((20,), 128, dtype=torch.int32, device=DEV)
    query = torch.randn(32, 128, generator=gen(3)).half().to(DEV)
    _, lse = ops.decode(query, kp, vp, ks, vs, valid, 4, 32, 1 / math.sqrt(128))
    w, _ = ops.attention_weights(query, kp, ks, valid, 4, 32, 1 / math.sqrt(128), lse=lse)
    torch.testing.assert_close(w.sum(-1), torch.full((8,), 4.0, device=DEV), rtol=5e-3, atol=0)
    w2, lse2 = ops.attention_weights(query, kp, ks, valid, 4, 32, 1 / math.sqrt(128))
    torch.testing.assert_close(w2.sum(-1), torch.full((8,), 4.0, device=DEV), rtol=1e-4, atol=0)
    torch.testing.assert_close(lse, lse2, rtol=1e-3, atol=5e-3)


@pytest.mark.parametrize("geometry", [(128, 4, 32), (96, 4, 48)])
def test_weights_refuse_blocks_outside_the_pool(geometry):
    d, bits, group = geometry
    ops.read_device_status(DEV)
    kp, ks = key_pool(3, 16, 2, d, bits, group, 2)
    valid = torch.tensor([16, 99, -4], dtype=torch.int32, device=DEV)
    table = torch.tensor([0, 3, -1, 0], dtype=torch.int32, device=DEV)
    query = torch.randn(4, d, generator=gen(3)).half().to(DEV)
    w, _ = ops.attention_weights(query, kp, ks, valid, bits, group, 0.1, block_table=table)
    assert ops.read_device_status(DEV) == _native.DEV_BAD_BLOCK
    assert (w[:, 16:48] == 0).all() and torch.equal(w[:, :16], w[:, 48:]) and (w[:, :16] > 0).all()
    ops.attention_weights(query, kp, ks, valid, bits, group, 0.1)
    assert ops.read_device_status(DEV) == _native.DEV_BAD_VALID


def test_weights_refusals():
    kp, ks = key_pool(2, 8, 2, 64, 4, 32, 2)
    valid = torch.full((2,), 8, dtype=torch.int32, device=DEV)
    q = torch.randn(4, 64, device=DEV)
    f = torch.zeros(4, device=DEV)
    w = torch.zeros(2, 16, device=DEV)
    call = lambda q=q, v=valid, b=4, gr=32, **kw: ops.attention_weights(q, kp, ks, v, b, gr, 0.1, **kw)  # noqa: E731
    for bad in (lambda: call(q=q.int()), lambda: call(q=q[0]), lambda: call(q=q[:3]),
                lambda: call(q=q[:, :32]), lambda: call(v=valid.long()), lambda: call(v=valid[:1]),
                lambda: call(b=2), lambda: call(gr=16), lambda: call(lse=f[:2]),
                lambda: call(lse=f.double()), lambda: call(visible=valid),
                lambda: call(block_table=valid.view(2, 1)), lambda: call(previous=w[:, :8]),
                lambda: call(out=w.t().contiguous().t()), lambda: call(previous=w.half())):
        with pytest.raises(ValueError):
            bad()


# ------------------------------------------------------------------------------------- evict


def stats(kvh, columns, n, seed, mixed=False, shared=False):
    g = gen(seed)
    w = torch.exp(2 * torch.randn(kvh, columns, generator=g)) * (torch.rand(kvh, columns, generator=g) > 0.3)
    order = torch.rand(kvh, n, generator=g).argsort(-1) if mixed else torch.arange(n).expand(kvh, n)
    if shared:
        order = order[:1].expand(kvh, n)
    pos = torch.full((kvh, columns), -1, dtype=torch.int32)
    pos[:, :n] = order
    return w, pos


def check_evict(w, pos, n, keep, nb, bt, pd, groups, *, table=None, sink=0, recent=0, shared=False,
                next_position=None, seed=0):
    kvh, columns = w.shape
    g = gen(seed)
    pool = [torch.randint(0, 256, (nb, bt, kvh, pd), generator=g, dtype=torch.uint8) for _ in "kv"]
    pool += [torch.rand(nb, bt, kvh, groups, generator=g).half() for _ in "kv"]
    valid = torch.full((nb,), -9, dtype=torch.int32)
    dev = [t.to(DEV) for t in pool]
    dvalid = valid.to(DEV)
    wd, pd_ = w.to(DEV), pos.to(DEV)
    new_w, new_p = ops.evict(wd, pd_, n, keep, *dev, dvalid, sink=sink, recent=recent, shared=shared,
                             next_position=next_position,
                             block_table=None if table is None else table.to(DEV))
    end = n if next_position is None else next_position
    source = orc.evict(w.numpy(), pos.numpy(), n, keep, sink, end - recent if recent else 1 << 40, shared)
    blocks = torch.arange(nb) if table is None else table.long()
    row = lambda i: blocks[i // bt] * bt + i % bt  # noqa: E731
    src = torch.from_numpy(source)
    to = row(torch.arange(keep)).expand(kvh, -1)
    heads = torch.arange(kvh).unsqueeze(-1)
    for got, t in zip(dev, pool):
        flat = t.flatten(0, 1)
        flat[to, heads] = flat[row(src), heads].clone()
        assert torch.equal(got.cpu(), t)
    ew, ep = torch.zeros_like(w), torch.full_like(pos, -1)
    ew[:, :keep], ep[:, :keep] = w.gather(1, src), pos.gather(1, src)
    np.testing.assert_array_equal(new_w.cpu().numpy(), ew.numpy())
    assert torch.equal(new_p.cpu(), ep)
    counts = (keep - bt * torch.arange(len(blocks))).clamp(0, bt).int()
    valid[blocks] = counts
    assert torch.equal(dvalid.cpu(), valid)
    assert torch.equal(wd.cpu().nan_to_num(7.0), w.nan_to_num(7.0)) and torch.equal(pd_.cpu(), pos)


@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("n, keep, bt, kvh, sink, recent, mixed", [
    (1, 1, 1, 1, 0, 0, False), (2, 1, 8, 2, 0, 0, False), (100, 99, 16, 2, 4, 8, False),
    (100, 1, 16, 3, 0, 1, True), (1000, 500, 40, 8, 4, 100, True), (4097, 2048, 128, 4, 0, 0, False),
    (9001, 8192, 128, 2, 16, 1000, True), (300, 300, 100, 2, 0, 0, False), (33, 32, 8, 1, 1, 31, False)])
def test_evict(n, keep, bt, kvh, sink, recent, mixed, shared):
    nb = -(-n // bt) + 1
    w, pos = stats(kvh, nb * bt + 3, n, n, mixed, shared)
    table = torch.randperm(nb, generator=gen(n)).int()
    check_evict(w, pos, n, keep, nb, bt, 64, 4, sink=sink, recent=recent, shared=shared)
    check_evict(w, pos, n, keep, nb, bt, 32, 4, sink=sink, recent=recent, shared=shared, table=table)


@pytest.mark.parametrize("pd, groups", [(64, 4), (16, 2), (6, 3), (32, 1), (128, 16), (5, 1), (12, 8)])
@pytest.mark.parametrize("shared", [False, True])
def test_evict_row_sizes(pd, groups, shared):
    w, pos = stats(3, 96, 90, 5, shared=shared)
    check_evict(w, pos, 90, 50, 6, 16, pd, groups, shared=shared, recent=3, sink=2)


@pytest.mark.parametrize("shared", [False, True])
def test_evict_ties_and_odd_weights(shared):
    w, pos = stats(2, 128, 128, 1, shared=shared)
    w[:] = 1.0  # all equal: the lowest places stay
    check_evict(w, pos, 128, 77, 8, 16, 16, 2, shared=shared)
    w[:, 3], w[:, 100], w[:, 101], w[:, 5] = math.inf, math.nan, -math.inf, -0.0
    w[:, 6], w[:, 90], w[:, 127], w[:, 20] = 0.0, -2.5, 3e38, 1e-42
    for keep in (1, 2, 64, 122, 123, 124, 125, 126, 127):
        check_evict(w, pos, 128, keep, 8, 16, 16, 2, shared=shared)
    w[:] = math.nan
    check_evict(w, pos, 128, 5, 8, 16, 16, 2, shared=shared)


def test_evict_next_position_and_strided_stats():
    w, pos = stats(4, 200, 150, 3)
    pos[:, :150] += 1000 * (pos[:, :150] > 20)  # tokens already gone
    check_evict(w, pos, 150, 60, 10, 16, 64, 4, sink=5, recent=30, next_position=1150)
    wide = torch.stack([w, w + 1], 1).reshape(4, 400)
    pool = [torch.zeros(10, 16, 4, 8, dtype=torch.uint8, device=DEV) for _ in "kv"] + [
        torch.zeros(10, 16, 4, 1, dtype=torch.float16, device=DEV) for _ in "kv"]
    valid = torch.zeros(10, dtype=torch.int32, device=DEV)
    a = ops.evict(wide.to(DEV)[:, :200], pos.to(DEV), 150, 60, *pool, valid)
    b = ops.evict(w.to(DEV), pos.to(DEV), 150, 60, *pool, valid)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_evict_long_cache():
    """More places than the select kernel keeps in shared memory; one KV head, one-byte rows."""
    n = 450_000
    w, pos = stats(1, n, n, 11)
    nb = -(-n // 128)
    dw = w.to(DEV)
    pool = [torch.arange(nb * 128, device=DEV).remainder(251).to(torch.uint8).view(nb, 128, 1, 1).clone()
            for _ in "kv"] + [torch.zeros(nb, 128, 1, 1, dtype=torch.float16, device=DEV) for _ in "kv"]
    valid = torch.zeros(nb, dtype=torch.int32, device=DEV)
    keep = 123_457
    new_w, new_p = ops.evict(dw, pos.to(DEV), n, keep, *pool, valid, recent=1000)
    order = np.lexsort((np.arange(n), -w[0].numpy().astype(np.float64), ~(np.arange(n) >= n - 1000)))
    kept = np.zeros(n, bool)
    kept[order[:keep]] = True
    source = np.arange(keep)
    source[~kept[:keep]] = keep + np.nonzero(kept[keep:])[0]
    np.testing.assert_array_equal(new_p[0, :keep].cpu().numpy(), source)
    np.testing.assert_array_equal(new_w[0, :keep].cpu().numpy(), w[0].numpy()[source])
    np.testing.assert_array_equal(pool[0].flatten()[:keep].cpu().numpy(), source % 251)
    np.testing.assert_array_equal(pool[0].flatten()[keep:].cpu().numpy(), np.arange(keep, nb * 128) % 251)


@pytest.mark.parametrize("n, shared", [(150_000, True), (400_003, False), (400_000, True)])
def test_evict_long_caches_by_head(n, shared):
    """Long caches of two heads, with and without vector accesses, against a sort."""
    nb = -(-n // 64)
    w, pos = stats(2, nb * 64, n, n, mixed=True, shared=shared)
    pool = [torch.randint(0, 256, (nb, 64, 2, 4), generator=gen(1), dtype=torch.uint8) for _ in "kv"] + [
        torch.rand(nb, 64, 2, 1, generator=gen(2)).half() for _ in "kv"]
    dev = [t.to(DEV) for t in pool]
    valid = torch.zeros(nb, dtype=torch.int32, device=DEV)
    keep = n // 3
    new_w, new_p = ops.evict(w.to(DEV), pos.to(DEV), n, keep, *dev, valid, sink=3, recent=77, shared=shared)
    total = w[:, :n].numpy().astype(np.float64).sum(0).astype(np.float32)
    for h in range(2):
        rank = total if shared else w[h, :n].numpy()
        p = pos[h, :n].numpy()
        order = np.lexsort((np.arange(n), -rank.astype(np.float64), ~((p < 3) | (p >= n - 77))))
        kept = np.zeros(n, bool)
        kept[order[:keep]] = True
        source = np.arange(keep)
        source[~kept[:keep]] = keep + np.nonzero(kept[keep:])[0]
        np.testing.assert_array_equal(new_p[h, :keep].cpu().numpy(), p[source])
        np.testing.assert_array_equal(new_w[h, :keep].cpu().numpy(), w[h].numpy()[source])
        assert (new_p[h, keep:] == -1).all() and (new_w[h, keep:] == 0).all()
        for got, t in zip(dev, pool):
            flat = t.flatten(0, 1)[:, h].numpy()
            now = got.flatten(0, 1)[:, h].cpu().numpy()
            np.testing.assert_array_equal(now[:keep], flat[source])
            np.testing.assert_array_equal(now[keep:], flat[keep:])


@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("n", [4095, 4097, 8193, 16385, 32768, 32769, 50_001, 65_537, 131_071, 131_073])
def test_evict_lengths(n, shared):
    """To either side of the lengths at which the selection takes more CTAs or more places a thread."""
    test_evict_long_caches_by_head(n, shared)


@pytest.mark.parametrize("n", [8192, 12_000, 16_385, 40_000])
def test_evict_many_heads(n):
    w, pos = stats(40, -(-n // 64) * 64, n, n)
    check_evict(w, pos, n, n // 2, -(-n // 64), 64, 4, 1, recent=9)


def test_evict_refuses_blocks_outside_the_pool():
    ops.read_device_status(DEV)
    w, pos = stats(1, 32, 32, 3)
    w[0] = torch.arange(32)
    pool = [torch.arange(4 * 8, dtype=torch.uint8, device=DEV).view(4, 8, 1, 1).clone() for _ in "kv"] + [
        torch.zeros(4, 8, 1, 1, dtype=torch.float16, device=DEV) for _ in "kv"]
    valid = torch.full((4,), 8, dtype=torch.int32, device=DEV)
    table = torch.tensor([0, 4, 2, -1], dtype=torch.int32, device=DEV)
    ops.evict(w.to(DEV), pos.to(DEV), 32, 16, *pool, valid, block_table=table)
    assert ops.read_device_status(DEV) == _native.DEV_BAD_BLOCK
    # places 0..7 take 16..23 (block 2); 8..15 (refused) would have taken 24..31 (refused)
    rows = pool[0].flatten().cpu()
    assert rows[:8].tolist() == list(range(16, 24)) and rows[8:].tolist() == list(range(8, 32))
    assert valid.cpu().tolist() == [8, 8, 0, 8]


def test_evict_refusals():
    w, pos = (t.to(DEV) for t in stats(2, 16, 16, 3))
    pool = [torch.zeros(2, 8, 2, 16, dtype=torch.uint8, device=DEV) for _ in "kv"] + [
        torch.zeros(2, 8, 2, 1, dtype=torch.float16, device=DEV) for _ in "kv"]
    valid = torch.zeros(2, dtype=torch.int32, device=DEV)
    call = lambda n=16, keep=8, w=w, pos=pos, valid=valid, **kw: ops.evict(w, pos, n, keep, *pool, valid, **kw)  # noqa: E731
    for bad in (lambda: call(n=17), lambda: call(n=0), lambda: call(keep=0), lambda: call(keep=17),
                lambda: call(sink=5, recent=4), lambda: call(sink=-1), lambda: call(w=w[:1]),
                lambda: call(w=w.double()), lambda: call(pos=pos.long()), lambda: call(pos=pos[:, :8]),
                lambda: call(w=w[:, :8], pos=pos[:, :8]), lambda: call(valid=valid[:1]),
                lambda: call(block_table=valid[:1]), lambda: call(w=w[:1].expand(2, 16))):
        with pytest.raises(ValueError):
            bad()


# ------------------------------------------------------------------------- together, streams, graphs


def dense(q, k, v, scale):
    """Attention weights and output in 64 bits of one query over per-head keys [KVH, n, D]."""
    qh = q.reshape(k.shape[0], -1, q.shape[-1]).double()
    p = torch.softmax(torch.einsum("hgd,hnd->hgn", qh, k) * scale, -1)
    return p.sum(1), torch.einsum("hgn,hnd->hgd", p, v).reshape(q.shape)


@pytest.mark.parametrize("bits, shared", [(4, False), (4, True), (2, False)])
def test_a_sequence_through_the_cache(bits, shared):
    """Prompt, observation window, decode steps, eviction, more steps: each step's output and the
    running weights against 64-bit attention over the tokens that each head still keeps."""
    spec = CacheSpec(layers=1, kv_heads=4, head_dim=128, block_tokens=32, bits=bits, group_size=32)
    emb = RotaryEmbedding(128, scaling="smooth", factor=4.0, original_length=256)
    cache = DeviceKVCache(spec, 12, DEV, rotary=emb)
    g = gen(bits)
    scale = 1 / math.sqrt(128)
    f = emb.frequencies().numpy()
    held_k, held_v = [], []  # per token [KVH, D] float64, what the cache holds

    def add(t):
        k, v = (torch.randn(t, 4, 128, generator=g).half() for _ in "kv")
        kv, vv = cache.append(k.to(DEV), v.to(DEV), values=True)
        at = len(held_k) + np.arange(t)
        k32 = torch.from_numpy(orc.rotate(k.double().numpy(), at, f).astype(np.float32))
        for x, got, held in ((k32, kv, held_k), (v.float(), vv, held_v)):
            q = quantize_tensor(x, bits, 32)
            assert torch.equal(got.cpu(), dequantize_tensor(q, torch.float16))
            held += list(dequantize_tensor(q).double())

    def kept():
        pos = cache.positions[:, :cache.n_tokens].cpu().long()
        k, v = torch.stack(held_k), torch.stack(held_v)
        h = torch.arange(4).unsqueeze(-1)
        return k[pos, h], v[pos, h]

    running = torch.zeros(4, cache.capacity, dtype=torch.float64)
    add(201)
    window = torch.randn(8, 16, 128, generator=g).half()
    turned = emb.apply(window.to(DEV), torch.arange(193, 201, device=DEV)).cpu()
    cache.observe(window.to(DEV))
    k, v = kept()
    for i in range(8):
        running[:, :194 + i] += dense(turned[i], k[:, :194 + i], v[:, :194 + i], scale)[0]
    torch.testing.assert_close(cache.weights.cpu().double(), running, rtol=1e-4, atol=1e-7)
    for step in range(40):
        add(1)
        q = torch.randn(16, 128, generator=g).half()
        out, _ = cache.decode(q.to(DEV), observe=True)
        turned = emb.apply(q[None].to(DEV), torch.tensor([cache.next_position - 1], device=DEV))[0].cpu()
        w, o = dense(turned, *kept(), scale)
        torch.testing.assert_close(out.cpu().double(), o, atol=2e-3, rtol=1e-2)
        running[:, :cache.n_tokens] += w
        # the step's log-sum-exp is the decode kernel's (its parity tolerance, 5e-3)
        torch.testing.assert_close(cache.weights.cpu().double(), running, rtol=6e-3, atol=1e-6)
        running = cache.weights.cpu().double()
        if step % 10 == 9:
            n = cache.n_tokens
            source = torch.from_numpy(orc.evict(cache.weights.cpu().numpy(), cache.positions.cpu().numpy(),
                                                n, 150, 4, cache.next_position - 16, shared))
            pos = cache.positions.cpu()[:, :n].gather(1, source)
            cache.evict(150, sink=4, recent=16, shared=shared)
            assert cache.n_tokens == 150 and torch.equal(cache.positions[:, :150].cpu(), pos)
            running = torch.zeros_like(running)
            running[:, :150] = cache.weights.cpu().double()[:, :150]
            assert (cache.weights[:, 150:] == 0).all()
    cache.check()
    assert ops.read_device_status(DEV) == 0


def test_cache_refusals_and_from_pool():
    spec = CacheSpec(layers=1, kv_heads=2, head_dim=64, block_tokens=8, bits=4, group_size=32)
    cache = DeviceKVCache(spec, 2, DEV)
    x = torch.randn(17, 2, 64, device=DEV).half()
    with pytest.raises(ValueError, match="do not fit"):
        cache.append(x, x)
    with pytest.raises(ValueError, match="empty"):
        cache.decode(x[0])
    cache.append(x[:13], x[:13])
    q = torch.randn(4, 64, device=DEV).half()
    with pytest.raises(ValueError):
        cache.decode(q[None])
    with pytest.raises(ValueError):
        cache.observe(torch.randn(14, 4, 64, device=DEV))
    cache.evict(13)  # nothing to do
    pool = DeviceBlockPool(spec, cache.packed_k, cache.packed_v, cache.scales_k, cache.scales_v,
                           cache.valid_tokens)
    copy = DeviceKVCache.from_pool(pool, 13, extra_blocks=1)
    torch.testing.assert_close(copy.decode(q)[0], cache.decode(q)[0])
    with pytest.raises(ValueError, match="cannot hold"):
        DeviceKVCache.from_pool(pool, 8)
    copy.append(x[:8], x[:8])
    assert copy.n_tokens == 21 and copy.valid_tokens.tolist() == [8, 8, 5]
    copy.evict(10)
    with pytest.raises(ValueError, match="different tokens"):
        copy.evict(5, shared=True)
    with pytest.raises(ValueError, match="before evicting"):
        copy.observe(torch.randn(2, 4, 64, device=DEV))
    with pytest.raises(ValueError):
        DeviceKVCache(spec, 2, DEV, rotary=RotaryEmbedding(128))


def everything(seed, n=700, keep=300):
    """Inputs of one call of each operator, and a function that makes the calls into fixed buffers."""
    g = gen(seed)
    bt, kvh, d = 128, 8, 128
    pool = make_pool(6, bt, kvh, d, 4, 32)
    x = torch.randn(n, kvh, d, generator=g).half().to(DEV)
    slots = torch.arange(n, device=DEV)
    f = freqs(64).to(DEV)
    valid = torch.zeros(6, dtype=torch.int32, device=DEV)
    q = torch.randn(3, 32, d, generator=g).half().to(DEV)
    pos = torch.arange(6 * bt, dtype=torch.int32, device=DEV).expand(kvh, -1).contiguous()

    def call():
        turned = ops.rotary(q, slots[:3], f)
        held = ops.append(x, x, slots, *pool, 4, 32, positions=slots, frequencies=f,
                          valid_tokens=valid, values=True)
        w, lse = ops.attention_weights(turned, pool[0], pool[2], valid, 4, 32, 0.1)
        w2, _ = ops.attention_weights(turned, pool[0], pool[2], valid, 4, 32, 0.1, lse=lse, previous=w)
        valid2, pool2 = valid.clone(), [t.clone() for t in pool]
        new = ops.evict(w2, pos, n, keep, *pool2, valid2, sink=4, recent=16)
        return [turned, *held, w, lse, w2, *new, valid2, *pool2]

    return call


def test_two_streams_and_repeats_are_bit_equal():
    calls = [everything(s) for s in (1, 2)]
    torch.cuda.synchronize()
    ref = [[t.clone() for t in c()] for c in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    for _ in range(5):
        got = []
        for s, c in zip(streams, calls):
            with torch.cuda.stream(s):
                got.append(c())
        torch.cuda.synchronize()
        for a, b in zip(ref, got):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_graphs_replayed_side_by_side():
    calls = [everything(s) for s in (3, 4)]
    ref = [[t.clone() for t in c()] for c in calls]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for c in calls:
            c()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for c in calls:  # both captured on one stream: they share no scratch
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs.append(c())
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in calls]
    for _ in range(3):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(ref, outs):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_offsets_beyond_32_bits():
    """A pool of more than 2^32 bytes of codes: rows at its end are written, scored and moved."""
    nb, bt, kvh, d = 70_000, 128, 8, 128
    pool = [torch.zeros(nb, bt, kvh, d // 2, dtype=torch.uint8, device=DEV),
            torch.zeros(nb, bt, kvh, d // 2, dtype=torch.uint8, device=DEV),
            torch.zeros(nb, bt, kvh, 4, dtype=torch.float16, device=DEV),
            torch.zeros(nb, bt, kvh, 4, dtype=torch.float16, device=DEV)]
    assert pool[0].numel() > 2**32
    valid = torch.zeros(nb, dtype=torch.int32, device=DEV)
    x = torch.randn(200, kvh, d, generator=gen(1)).half()
    slots = torch.arange(200) + (nb - 2) * bt
    ops.append(x.to(DEV), x.to(DEV), slots.to(DEV), *pool, 4, 32, valid_tokens=valid)
    packed, scales, _ = quantized(x.float(), 4, 32)
    tail = [t[-2:].flatten(0, 1)[:200] for t in pool]
    assert torch.equal(tail[0].cpu(), packed) and torch.equal(tail[3].cpu(), scales)
    table = torch.tensor([nb - 2, nb - 1], dtype=torch.int32, device=DEV)
    q = torch.randn(32, d, generator=gen(2)).half().to(DEV)
    got = ops.attention_weights(q, pool[0], pool[2], valid, 4, 32, 0.1, block_table=table)
    small = [t[-2:].contiguous() for t in pool]
    ref = ops.attention_weights(q, small[0], small[2], valid[-2:].contiguous(), 4, 32, 0.1)
    assert torch.equal(got[0], ref[0])
    pos = torch.arange(256, dtype=torch.int32, device=DEV).expand(kvh, -1).contiguous()
    a = ops.evict(got[0], pos, 200, 100, *pool, valid, block_table=table)
    b = ops.evict(ref[0], pos, 200, 100, *small, torch.zeros(2, dtype=torch.int32, device=DEV))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    assert all(torch.equal(t[-2:], s) for t, s in zip(pool, small))
    assert valid[-2:].tolist() == [100, 0]
