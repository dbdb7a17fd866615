"""Cache-maintenance operators on a B200 at the edges of their ranges: uneven head counts with long tile
tables, numbers that are not numbers where a query sees them, scales at the end of FP32, scratch sizes,
and DeviceKVCache's failures and captures."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from kvssd_b200 import CacheSpec, DeviceBlockPool, DeviceKVCache, _native, ops
from kvssd_b200.quant import quantize_tensor
from oracle import cache_oracle as orc
from test_gpu_cache_ops import check_weights

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def gen(seed):
    return torch.Generator().manual_seed(seed)


def key_pool(nb, bt, kvh, d, bits, group, seed):
    q = quantize_tensor(torch.randn(nb, bt, kvh, d, generator=gen(seed)) * 1.5, bits, group)
    return q.packed.to(DEV), q.scales.to(DEV)


# ------------------------------------------------------------------------------------------ rotary


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_into_views_that_leave_places_out(interleaved):
    """Every second head of an odd number of heads, every second token, heads first: `out` does not overlap
    itself, however close the rows lie; what lies between them stays."""
    f = (10000.0 ** (-torch.arange(16, dtype=torch.float64) / 16)).to(DEV)
    x = torch.randn(6, 5, 64, generator=gen(1)).half().to(DEV)
    views = [lambda t: t[:, ::2], lambda t: t[::2], lambda t: t[::5, 1:4], lambda t: t[:1, ::4], lambda t: t[:, 2:3],
             lambda t: t.transpose(0, 1)[::2], lambda t: t.view(30, 1, 64)[::29], lambda t: t.view(1, 30, 64)[:, ::29]]
    for view in views:
        want = view(x).contiguous()
        positions = torch.arange(want.shape[0], device=DEV) + 9
        want = ops.rotary(want, positions, f, interleaved=interleaved)
        out = torch.full_like(x, 7.0)
        assert ops.rotary(view(x), positions, f, interleaved=interleaved, out=view(out)).shape == want.shape
        rest = out.clone()
        view(rest).fill_(7.0)
        assert torch.equal(view(out), want) and (rest == 7.0).all()
        mine = x.clone()
        ops.rotary(view(mine), positions, f, interleaved=interleaved, out=view(mine))
        assert torch.equal(view(mine), want)
    flat = torch.empty(600, dtype=torch.float16, device=DEV)
    x = x[:2, :3]
    positions = positions[:2]
    for strides in ((64, 0), (0, 64), (63, 200), (200, 63), (191, 64), (64, 127), (128, 64)):
        with pytest.raises(ValueError, match="overlap"):
            ops.rotary(x, positions, f, out=flat.as_strided((2, 3, 64), (*strides, 1)))


# ------------------------------------------------------------------------------- attention weights


@pytest.mark.parametrize("kvh, places, d, bits, group, dtype", [
    (60, 9_000, 64, 4, 32, torch.float16), (60, 9_000, 64, 2, 16, torch.float32),
    (20, 23_000, 96, 4, 32, torch.bfloat16), (20, 23_000, 64, 4, 32, torch.float32),
    (9, 30_000, 64, 2, 32, torch.float16), (14, 45_000, 64, 4, 16, torch.float16),
    (12, 44_400, 128, 4, 32, torch.float16), (7, 90_000, 64, 2, 32, torch.bfloat16)])
def test_weights_step_many_short_blocks_of_uneven_heads(kvh, places, d, bits, group, dtype):
    """Head counts that leave warps of a CTA over, with more than 256 tiles a CTA: every place gets what
    its pool block gets in a short call over the pool, bit for bit."""
    pool = 97
    kp, ks = key_pool(pool, 1, kvh, d, bits, group, kvh)
    valid = torch.ones(pool, dtype=torch.int32, device=DEV)
    valid[5] = 0
    query = torch.randn(kvh, d, generator=gen(1)).to(dtype).to(DEV)
    lse = torch.linspace(-1.0, 2.0, kvh, device=DEV)
    scale = 1 / math.sqrt(d)
    table = torch.randint(0, pool, (places,), generator=gen(places)).int().to(DEV)
    once, _ = ops.attention_weights(query, kp, ks, valid, bits, group, scale, lse=lse)
    assert (once[:, 5] == 0).all() and (once[:, 6:] > 0).all()
    many, _ = ops.attention_weights(query, kp, ks, valid, bits, group, scale, lse=lse, block_table=table)
    assert torch.equal(many, once[:, table.long()])
    assert ops.read_device_status(DEV) == 0


def check_nan(query, kp, ks, valid, bits, group, scale, visible=None):
    """NaN exactly where the 64-bit form has it; elsewhere scores of order one, whose FP32 sums of up to
    256 products are off by less than 2^-13: 1e-3 of a weight, absolutely of a log-sum-exp."""
    out, lse = ops.attention_weights(query, kp, ks, valid, bits, group, scale, visible=visible)
    cpu = lambda t: None if t is None else t.cpu().numpy()  # noqa: E731
    w, full, _ = orc.attention_weights(query.double().cpu().numpy(), cpu(kp), cpu(ks), cpu(valid), bits, group,
                                       scale, visible=cpu(visible))
    for got, want in ((out.double().cpu().numpy(), w), (lse.double().cpu().numpy(), full)):
        assert (np.isnan(got) == np.isnan(want)).all()
        np.testing.assert_allclose(got, want, rtol=1e-3, atol=1e-3 if want is full else 1e-30)
    return out, lse


NAN_SHAPES = [  # gqa, d, bits, group, queries: forms for any shape, for steps, windows and long windows
    (2, 32, 4, 8, 2), (1, 80, 2, 40, 3), (12, 36, 4, 12, 5), (2, 128, 4, 32, 2), (3, 64, 2, 16, 2),
    (4, 128, 2, 32, 5), (4, 96, 4, 48, 6), (10, 128, 4, 32, 5), (10, 64, 2, 32, 4), (40, 256, 2, 64, 2)]


@pytest.mark.filterwarnings("ignore::RuntimeWarning")
@pytest.mark.parametrize("shape", NAN_SHAPES)
def test_weights_nan_scores_show(shape):
    """A NaN in a query or in a key's scale shows in all that sees it, whichever place it has among the
    keys, and in nothing else."""
    gqa, d, bits, group, queries = shape
    kvh, nb, bt = 2, 5, 40
    n = nb * bt
    kp, ks = key_pool(nb, bt, kvh, d, bits, group, 3)
    valid = torch.full((nb,), bt, dtype=torch.int32, device=DEV)
    clean = torch.randn(queries, kvh * gqa, d, generator=gen(4)).to(DEV)
    scale = 1 / math.sqrt(d)
    query = clean.clone()
    query[-1, gqa, 1] = math.nan  # the last query's first head of KV head 1
    _, lse = check_nan(query, kp, ks, valid, bits, group, scale)
    assert lse.isnan().sum() == 1
    seen = torch.full((queries,), n, dtype=torch.int32, device=DEV)
    seen[-1] = 70
    out, _ = check_nan(query, kp, ks, valid, bits, group, scale, visible=seen)
    assert out[1, :70].isnan().all() and not out[1, 70:].isnan().any() and not out[0].isnan().any()
    for place in (0, 32, 45, 63, n - 1):  # first, later and last places of a run of 32, of all
        broken = ks.clone()
        broken[place // bt, place % bt, 0, -1] = math.nan
        out, lse = check_nan(clean, kp, broken, valid, bits, group, scale)
        assert out[0].isnan().all() and not out[1].isnan().any()
        seen = torch.full((queries,), n, dtype=torch.int32, device=DEV)
        seen[0] = place  # the first query sees the places before it only
        check_nan(clean, kp, broken, valid, bits, group, scale, visible=seen)
    valid[-1] = bt - 1  # behind the valid rows it does not show
    out, lse = check_nan(clean, kp, broken, valid, bits, group, scale)
    assert not out.isnan().any() and not lse.isnan().any()


@pytest.mark.filterwarnings("ignore::RuntimeWarning")
@pytest.mark.parametrize("shape", [*NAN_SHAPES, (80, 128, 2, 32, 2)])
def test_weights_of_queries_that_add_nothing_beside_nan_keys(shape):
    """Queries given as -inf add nothing to any place, to one whose key's scale is NaN neither; nor does
    one that does not see that place."""
    gqa, d, bits, group, queries = shape
    kvh, nb, bt = 2, 5, 64
    kp, ks = key_pool(nb, bt, kvh, d, bits, group, 3)
    ks[2, 22, :, 0] = ks[4, 63] = math.nan
    valid = torch.full((nb,), bt, dtype=torch.int32, device=DEV)
    query = torch.randn(queries, kvh * gqa, d, generator=gen(4)).half().to(DEV)
    previous = torch.rand(kvh, nb * bt, generator=gen(5)).to(DEV)
    lse = torch.full((queries, kvh * gqa), -math.inf, device=DEV)
    call = lambda **kw: ops.attention_weights(query, kp, ks, valid, bits, group, 0.1, lse=lse,  # noqa: E731
                                              previous=previous, **kw)[0]
    assert torch.equal(call(), previous)
    lse[0, 0] = 3.0  # one row of KV head 0 that sees all
    out = call()
    assert torch.equal(out[1], previous[1])
    assert out[0].isnan().nonzero().flatten().tolist() == [150, nb * bt - 1]
    seen = torch.full((queries,), 150, dtype=torch.int32, device=DEV)  # one that sees the places before them
    out = call(visible=seen)
    assert torch.equal(out[1], previous[1]) and torch.equal(out[0, 150:], previous[0, 150:])
    assert (out[0, :150] > previous[0, :150]).all()


@pytest.mark.parametrize("nb, bt, kvh, gqa, d, bits, group, queries, odd", [
    (90, 40, 8, 1, 80, 4, 40, 2, False), (4000, 1, 2, 3, 32, 2, 8, 1, False), (60, 100, 4, 2, 36, 4, 12, 9, False),
    (40, 128, 8, 2, 128, 4, 32, 3, True), (70, 100, 2, 20, 64, 2, 32, 2, True),
    (3000, 1, 2, 40, 64, 4, 32, 1, False), (1500, 3, 1, 17, 96, 2, 32, 2, False), (2000, 2, 8, 2, 256, 2, 64, 30, False),
    (700, 4, 160, 1, 64, 4, 32, 33, False), (300, 7, 8, 1, 128, 4, 16, 12, False), (5, 16, 600, 1, 80, 4, 16, 1, False),
    (110, 40, 32, 1, 20, 4, 4, 256, False), (300, 16, 16, 1, 64, 4, 32, 512, True)])
def test_weights_parts_of_the_log_sum_exps(nb, bt, kvh, gqa, d, bits, group, queries, odd):
    """Computed log-sum-exps where blocks are so short that a CTA's run of places is, with more KV heads than
    CTAs fit the GPU, and with so many rows that a CTA takes several runs; `odd`: a pool off 16 bytes."""
    kp, ks = key_pool(nb, bt, kvh, d, bits, group, 8)
    if odd:
        far = torch.empty(kp.numel() + 1, dtype=torch.uint8, device=DEV)[1:].view(kp.shape)
        kp = far.copy_(kp)
    valid = torch.full((nb,), bt, dtype=torch.int32, device=DEV)
    valid[-1] = 1
    valid[nb // 3] = 0
    query = torch.randn(queries, kvh * gqa, d, generator=gen(5)).half().to(DEV)
    visible = (nb * bt - queries + 1 + torch.arange(queries)).int().to(DEV)
    got = ops.attention_weights(query, kp, ks, valid, bits, group, 0.1, visible=visible)
    check_weights(query, kp, ks, valid, bits, group, 0.1, visible=visible, got=got)


# ------------------------------------------------------------------------------------------ append


def make_pool(nb, bt, kvh, d, bits, group):
    return [torch.zeros(nb, bt, kvh, d * bits // 8, dtype=torch.uint8, device=DEV) for _ in "kv"] + [
        torch.zeros(nb, bt, kvh, d // group, dtype=torch.float16, device=DEV) for _ in "kv"]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bits", [2, 4])
@pytest.mark.parametrize("d, group, kvh", [(128, 32, 2), (64, 64, 3), (128, 16, 1), (20, 4, 2)])
def test_append_at_the_end_of_fp32(d, group, kvh, bits, dtype):
    """Groups whose largest element lies between 2^120 and the largest number of the type, and groups of the
    smallest: codes and scales (infinite in FP16 at the top) are the quantizer's."""
    top = torch.finfo(dtype).max
    tokens = 40
    x = torch.rand(tokens, kvh, d, generator=gen(bits)) * 2 - 1
    size = 2.0 ** torch.linspace(-149, 127.9, tokens - 4)
    x[4:] *= size[:, None, None]
    x[0] *= top
    x[1] *= top / 2
    x[1, :, 0::group] = top
    x[2] *= 2.0**125
    x[2, :, 1::group] = -(2.0**126)
    x[3] *= 2.0**126
    x[3, :, 1::group] = 2.0**126 * 1.0078125
    x = x.to(dtype)
    assert x.isfinite().all()
    pool = make_pool(5, 8, kvh, d, bits, group)
    ops.append(x.to(DEV), (-x).to(DEV), torch.arange(tokens, device=DEV), *pool, bits, group)
    for i, y in enumerate((x, -x)):
        q = quantize_tensor(y.float(), bits, group)
        assert torch.equal(pool[i].flatten(0, 1).cpu(), q.packed)
        assert torch.equal(pool[2 + i].flatten(0, 1).cpu(), q.scales)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("tokens, kvh, d, bits, group, pairs", [
    (37, 2, 128, 4, 32, 64), (300, 8, 128, 2, 32, 32), (9, 3, 20, 4, 4, 7), (1200, 1, 64, 4, 16, 32)])
def test_append_with_a_magnitude(tokens, kvh, d, bits, group, pairs, dtype, interleaved):
    """Keys rotated with cos and sin times a magnitude (taken in FP32, as the entry point does)."""
    magnitude = float(np.float32(0.1 * math.log(4.0) + 1.0))
    g = gen(tokens + d)
    key, value = [(torch.randn(tokens, kvh, d, generator=g) * 2).to(dtype) for _ in "kv"]
    positions = torch.arange(tokens) * 7 + 54_321
    f = 10000.0 ** (-torch.arange(pairs, dtype=torch.float64) / pairs)
    nb = -(-tokens // 16)
    pool = make_pool(nb, 16, kvh, d, bits, group)
    ops.append(key.to(DEV), value.to(DEV), torch.arange(tokens, device=DEV), *pool, bits, group,
               positions=positions.to(DEV), frequencies=f.to(DEV), interleaved=interleaved,
               magnitude=magnitude)
    turned = orc.rotate(key.double().numpy(), positions.numpy(), f.numpy(), interleaved, magnitude)
    for i, y in enumerate((torch.from_numpy(turned.astype(np.float32)), value.float())):
        q = quantize_tensor(y, bits, group)
        assert torch.equal(pool[i].flatten(0, 1)[:tokens].cpu(), q.packed)
        assert torch.equal(pool[2 + i].flatten(0, 1)[:tokens].cpu(), q.scales)


# ------------------------------------------------------------------------------------------- evict


def test_evict_into_given_tensors():
    weights = torch.rand(2, 40, generator=gen(1)).to(DEV)
    positions = torch.arange(40, dtype=torch.int32, device=DEV).expand(2, 40).contiguous()
    pool = [torch.randint(0, 256, (5, 8, 2, 16), generator=gen(2), dtype=torch.uint8).to(DEV) for _ in "kv"] + [
        torch.rand(5, 8, 2, 1, generator=gen(3)).half().to(DEV) for _ in "kv"]
    call = lambda out=None: ops.evict(weights, positions, 37, 20, *(t.clone() for t in pool),  # noqa: E731
                                      torch.zeros(5, dtype=torch.int32, device=DEV), sink=2, out=out)
    want = call()
    wide = torch.full((4, 2, 40), 9, dtype=torch.int32, device=DEV)
    out = wide[1].view(torch.float32), wide[2]
    got = call(out)
    assert got[0] is out[0] and got[1] is out[1]
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert (wide[0] == 9).all() and (wide[3] == 9).all()
    spare = torch.empty_like(weights), torch.empty_like(positions)
    for bad in ((weights, spare[1]), (spare[0], positions), (spare[0].double(), spare[1]), (spare[0], spare[1].long()),
                (spare[0][:, :39], spare[1]), (spare[0], spare[1][:1]), (spare[0].cpu(), spare[1])):
        with pytest.raises(ValueError):
            call(bad)


# ------------------------------------------------------------------------------------ DeviceKVCache


SPEC = CacheSpec(layers=1, kv_heads=2, head_dim=64, block_tokens=8, bits=4, group_size=32)


def small_cache(tokens=13, blocks=4, rotary=None):
    cache = DeviceKVCache(SPEC, blocks, DEV, rotary)
    x = torch.randn(tokens, 2, 64, generator=gen(tokens)).half().to(DEV)
    cache.append(x, x)
    return cache


@pytest.mark.parametrize("pooled", [False, True])
def test_decode_captured_behind_decodes_on_the_same_stream(pooled):
    """The reads of the status word that earlier decodes left outstanding do not disturb a capture."""
    holder = small_cache()
    if pooled:
        holder = DeviceBlockPool(SPEC, *(t[:2] for t in (holder.packed_k, holder.packed_v, holder.scales_k,
                                                         holder.scales_v, holder.valid_tokens)))
    query = torch.randn(4, 64, generator=gen(2)).half().to(DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            ref = holder.decode(query)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = holder.decode(query)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out[0], ref[0]) and torch.equal(out[1], ref[1])
    with torch.cuda.stream(side):
        holder.check()


def status_word():
    """The status word of the current stream's workspace, as the kernels see it."""
    return ops._workspaces.get(DEV, torch.cuda.current_stream(DEV), 2048)[:4].view(torch.int32)


def test_cache_check_reports_a_failed_window():
    """A window whose wait gave up has set its bit and left NaN; check() raises, and clears it."""
    ops.read_device_status(DEV)
    cache = small_cache()
    query = torch.randn(3, 4, 64, generator=gen(1)).half().to(DEV)
    status_word().fill_(_native.DEV_STREAM_TIMEOUT)
    cache.observe(query)
    with pytest.raises(ops.DeviceFailure, match="gave up"):
        cache.check()
    cache.check()
    # flagged by a call that arms no read of its own
    status_word().fill_(_native.DEV_BAD_BLOCK)
    with pytest.raises(ops.DeviceFailure, match="outside the pool"):
        cache.check()
    assert ops.read_device_status(DEV) == 0


@pytest.mark.parametrize("call", ["observe", "evict"])
def test_cache_raises_a_known_failure_before_the_next_call(call):
    ops.read_device_status(DEV)
    cache = small_cache()
    query = torch.randn(3, 4, 64, generator=gen(1)).half().to(DEV)
    status_word().fill_(_native.DEV_STREAM_TIMEOUT)
    cache.observe(query)
    torch.cuda.synchronize()
    before = [t.clone() for t in (cache.packed_k, cache.weights, cache.positions)]
    with pytest.raises(ops.DeviceFailure, match=call):
        cache.evict(5) if call == "evict" else cache.observe(query)
    assert cache.n_tokens == 13
    assert all(torch.equal(a, b) for a, b in zip(before, (cache.packed_k, cache.weights, cache.positions)))
    cache.evict(5)
    cache.check()
    assert cache.n_tokens == 5


def test_a_graph_flags_in_a_workspace_that_has_been_replaced():
    """A captured call's status word outlives the workspace that held it; its flag is still read."""
    pool = [torch.zeros(2, 4, 1, 16, dtype=torch.uint8, device=DEV) for _ in "kv"] + [
        torch.zeros(2, 4, 1, 1, dtype=torch.float16, device=DEV) for _ in "kv"]
    x = torch.randn(2, 1, 32, generator=gen(1)).to(DEV)
    slots = torch.tensor([1, 3], device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.append(x, x, slots, *pool, 4, 32)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        ops.append(x, x, slots, *pool, 4, 32)
    with torch.cuda.stream(side):
        held = ops._workspaces.get(DEV, side, 2048)
        ops._workspaces.get(DEV, side, 4 * held.numel())
    del held
    torch.cuda.synchronize()
    slots[1] = 8  # behind the pool
    graph.replay()
    torch.cuda.synchronize()
    assert ops.read_device_status(DEV, stream=side) == _native.DEV_BAD_BLOCK
    assert ops.read_device_status(DEV, stream=side) == 0
    graph.replay()
    assert ops.read_device_status_all(DEV) & _native.DEV_BAD_BLOCK
    assert ops.read_device_status_all(DEV) == 0


def test_a_captured_decode_adds_to_the_weights_of_a_cache_that_evicted_since():
    """The buffers of a cache stay where they are: a graph captured before an eviction reads and adds to
    what the cache holds after it."""
    cache = small_cache()
    query = torch.randn(4, 64, generator=gen(3)).half().to(DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cache.decode(query, observe=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out, lse = cache.decode(query, observe=True)
    torch.cuda.synchronize()
    addresses = [t.data_ptr() for t in (cache.weights, cache.positions)]
    cache.evict(5, sink=2, recent=1)
    assert [t.data_ptr() for t in (cache.weights, cache.positions)] == addresses
    assert (cache.weights[:, 5:] == 0).all() and (cache.positions[:, 5:] == -1).all()
    assert (cache.positions[:, :5] >= 0).all()
    before = cache.weights.clone()
    graph.replay()
    torch.cuda.synchronize()
    added, own = ops.attention_weights(query, cache.packed_k, cache.scales_k, cache.valid_tokens, 4, 32, 1 / 8)
    torch.testing.assert_close(cache.weights - before, added, rtol=1e-2, atol=1e-3)  # lse: the decode's
    torch.testing.assert_close(lse, own, rtol=1e-3, atol=5e-3)
    assert (cache.weights[:, 5:] == 0).all()
    with torch.cuda.stream(side):
        cache.check()


def test_cache_calls_that_move_counts_refuse_a_capture():
    cache = small_cache()
    x = torch.randn(1, 2, 64, generator=gen(3)).half().to(DEV)
    query = torch.randn(4, 64, generator=gen(3)).half().to(DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ref = cache.decode(query)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        with pytest.raises(RuntimeError, match="cannot be captured"):
            cache.append(x, x)
        with pytest.raises(RuntimeError, match="cannot be captured"):
            cache.evict(5)
        out = cache.decode(query)
    assert cache.n_tokens == cache.next_position == 13
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out[0], ref[0]) and torch.equal(out[1], ref[1])
    cache.append(x, x)
    assert cache.n_tokens == 14


def test_status_of_a_device_given_without_its_index():
    """"cuda" is the current device: its flags are found and cleared."""
    ops.read_device_status(DEV)
    for read in (ops.read_device_status, ops.read_device_status_all):
        status_word().fill_(_native.DEV_BAD_BLOCK)
        assert read("cuda") == _native.DEV_BAD_BLOCK and read("cuda") == 0 and read(DEV) == 0
    assert ops.status_watch(torch.device("cuda")) is ops.status_watch(DEV)


def test_a_graph_of_a_fresh_stream_flags_what_it_refuses():
    """Captured on the stream that a graph brings along, which has run nothing: a slot behind the pool is
    reported all the same, of every replay."""
    pool = [torch.zeros(2, 4, 1, 16, dtype=torch.uint8, device=DEV) for _ in "kv"] + [
        torch.zeros(2, 4, 1, 1, dtype=torch.float16, device=DEV) for _ in "kv"]
    x = torch.randn(2, 1, 32, generator=gen(1)).to(DEV)
    slots = torch.tensor([1, 3], device=DEV)
    ops.append(x, x, slots, *pool, 4, 32)  # elsewhere
    torch.cuda.synchronize()
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=stream):
        ops.append(x, x, slots, *pool, 4, 32)
    assert ops.read_device_status_all(DEV) == 0
    graph.replay()
    assert ops.read_device_status_all(DEV) == 0
    slots[1] = 8
    for _ in range(2):
        graph.replay()
        assert ops.read_device_status_all(DEV) == _native.DEV_BAD_BLOCK
    assert ops.read_device_status_all(DEV) == 0
