"""DeviceKVCache: one layer's packed KV cache that grows, is read, and gives up its least used tokens.

Where DeviceBlockPool holds a finished layer, this holds the cache of a running sequence: tokens
are appended (their keys rotated and both quantized by one kernel), a decode step attends over
them and may add the weight each got to its running sum, and eviction keeps the tokens of the
largest sums. Everything stays on the device; a step makes no host synchronisation. The reference
has no counterpart (its cache is written once and read, src/kvssd/store.py:27-67, and its
selectors go by block order, src/kvssd/selectors.py:11-28).
"""

from __future__ import annotations

import math

import torch

from . import ops
from .format import CacheSpec
from .pool import DeviceBlockPool
from .rotary import RotaryEmbedding


class DeviceKVCache:
    """Cache of up to ``blocks * spec.block_tokens`` tokens of one layer on a CUDA device.

    ``n_tokens`` places are in use; place i is row i % block_tokens of block i // block_tokens.
    ``weights`` fp32 and ``positions`` int32 [kv_heads, places] hold each place's accumulated
    attention weight and the position of the token that each KV head keeps there.

    The counts live on the host. A captured ``decode`` or ``observe`` keeps the blocks and positions it
    was captured with; ``append`` and ``evict``, which a replay would repeat on the same places, refuse
    to be captured (a graph appends with ops.append, whose slots and positions lie on the device)."""

    def __init__(self, spec: CacheSpec, blocks: int, device: torch.device | str,
                 rotary: RotaryEmbedding | None = None):
        spec.validate()
        if blocks < 1:
            raise ValueError("at least one block is required")
        if rotary is not None and rotary.head_dim != spec.head_dim:
            raise ValueError(f"rotary head_dim {rotary.head_dim} differs from the cache's {spec.head_dim}")
        device = torch.device(device)
        if device.type != "cuda":
            raise RuntimeError(f"DeviceKVCache needs a CUDA device, got {device}")
        if device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        self.spec, self.device, self.rotary = spec, device, rotary
        codes = (blocks, spec.block_tokens, spec.kv_heads, spec.packed_dim)
        scales = (blocks, spec.block_tokens, spec.kv_heads, spec.groups)
        # zeros: decode kernels may read the scales of rows behind the valid count
        self.packed_k = torch.zeros(codes, dtype=torch.uint8, device=device)
        self.packed_v = torch.zeros(codes, dtype=torch.uint8, device=device)
        self.scales_k = torch.zeros(scales, dtype=torch.float16, device=device)
        self.scales_v = torch.zeros(scales, dtype=torch.float16, device=device)
        self.valid_tokens = torch.zeros(blocks, dtype=torch.int32, device=device)
        # one buffer, so that what an eviction leaves is copied back at once; a second one at the first
        self._stats = [torch.zeros((2, spec.kv_heads, self.capacity), dtype=torch.int32, device=device)]
        self._weights, self._positions = self._parts(self._stats[0])
        self._positions.fill_(-1)
        self._places = torch.arange(self.capacity, dtype=torch.int32, device=device)
        self.n_tokens = 0
        self.next_position = 0
        self._own_choices = False  # a per-head eviction has run

    @classmethod
    def from_pool(cls, pool: DeviceBlockPool, n_tokens: int, extra_blocks: int = 0,
                  rotary: RotaryEmbedding | None = None) -> "DeviceKVCache":
        """A cache that starts with a copy of ``pool``'s blocks, which hold ``n_tokens`` tokens in
        order (every block but the last full), with room for ``extra_blocks`` more."""
        if extra_blocks < 0:
            raise ValueError("extra_blocks must be non-negative")
        bt, n = pool.spec.block_tokens, pool.n_blocks
        if not (n - 1) * bt < n_tokens <= n * bt:
            raise ValueError(f"{n} blocks of {bt} tokens cannot hold {n_tokens} tokens in order")
        cache = cls(pool.spec, n + extra_blocks, pool.device, rotary)
        for name in ("packed_k", "packed_v", "scales_k", "scales_v", "valid_tokens"):
            getattr(cache, name)[:n].copy_(getattr(pool, name))
        cache.positions[:, :n_tokens] = cache._places[:n_tokens]
        cache.n_tokens = cache.next_position = n_tokens
        return cache

    @staticmethod
    def _parts(stats: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        return stats[0].view(torch.float32), stats[1]

    @property
    def weights(self) -> torch.Tensor:
        return self._weights

    @property
    def positions(self) -> torch.Tensor:
        return self._positions

    @property
    def capacity(self) -> int:
        return self.packed_k.shape[0] * self.spec.block_tokens

    @property
    def used_blocks(self) -> int:
        return -(-self.n_tokens // self.spec.block_tokens)

    def append(self, key: torch.Tensor, value: torch.Tensor, *,
               values: bool = False) -> tuple[torch.Tensor, torch.Tensor] | None:
        """Adds the tokens of ``key`` and ``value`` [tokens, kv_heads, head_dim] (keys not yet rotated)
        at the next positions; see ops.append."""
        self._not_captured("append")
        tokens = key.shape[0]
        n = self.n_tokens
        if n + tokens > self.capacity:
            raise ValueError(f"{tokens} more tokens do not fit: {n} of {self.capacity} places are used")
        at = self.next_position
        positions = torch.arange(at, at + tokens, dtype=torch.int32, device=self.device)
        turn = {}
        if self.rotary is not None:
            turn = dict(positions=positions, frequencies=self.rotary.on(self.device),
                        interleaved=self.rotary.interleaved, magnitude=self.rotary.magnitude)
        held = ops.append(key, value, self._places[n:n + tokens], self.packed_k, self.packed_v,
                          self.scales_k, self.scales_v, self.spec.bits, self.spec.group_size,
                          valid_tokens=self.valid_tokens, values=values, **turn)
        self.positions[:, n:n + tokens] = positions
        self.n_tokens, self.next_position = n + tokens, at + tokens
        return held

    def _not_captured(self, call: str) -> None:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError(f"DeviceKVCache.{call} moves counts on the host and cannot be captured in a graph")

    def _in_use(self):
        if self.n_tokens == 0:
            raise ValueError("the cache is empty")
        b = self.used_blocks
        return b, self.packed_k[:b], self.scales_k[:b], self.valid_tokens[:b]

    def _rotated(self, query: torch.Tensor) -> torch.Tensor:
        """Queries [T, query_heads, head_dim] of the last T tokens."""
        if self.rotary is None:
            return query
        end = self.next_position
        positions = torch.arange(end - query.shape[0], end, dtype=torch.int32, device=self.device)
        return self.rotary.apply(query, positions)

    def _scale(self, sm_scale: float | None) -> float:
        return 1.0 / math.sqrt(self.spec.head_dim) if sm_scale is None else sm_scale

    def decode(self, query: torch.Tensor, sm_scale: float | None = None,
               observe: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
        """(out fp32 [query_heads, head_dim], lse fp32 [query_heads]) of the last token's query
        [query_heads, head_dim] (not yet rotated) over the cache; ``observe`` adds the weight each
        place got to ``weights``. Asynchronous; failures surface as DeviceBlockPool's do."""
        if query.ndim != 2:
            raise ValueError("query must be [query_heads, head_dim]")
        b, packed_k, scales_k, valid = self._in_use()
        query = self._rotated(query.unsqueeze(0)).squeeze(0)
        scale = self._scale(sm_scale)
        watch = ops.status_watch(self.device)
        watch.poll("DeviceKVCache.decode (an earlier call)")
        out, lse = ops.decode(query, packed_k, self.packed_v[:b], scales_k, self.scales_v[:b], valid,
                              self.spec.bits, self.spec.group_size, scale)
        if observe:
            weights = self.weights[:, :b * self.spec.block_tokens]
            ops.attention_weights(query, packed_k, scales_k, valid, self.spec.bits,
                                  self.spec.group_size, scale, lse=lse, previous=weights, out=weights)
        watch.arm("DeviceKVCache.decode")
        return out, lse

    def observe(self, query: torch.Tensor, sm_scale: float | None = None) -> torch.Tensor:
        """Adds the weights that the last T tokens' queries [T, query_heads, head_dim] (not yet
        rotated) give the cache, each seeing the places up to its own token; returns their
        log-sum-exps [T, query_heads]. For a prompt, before anything has been evicted. Asynchronous, as
        ``decode`` is; after a failure ``weights`` hold NaN."""
        if query.ndim != 3 or not 1 <= query.shape[0] <= self.n_tokens:
            raise ValueError("query must be [T, query_heads, head_dim] of the last T tokens")
        if self.next_position != self.n_tokens:
            raise ValueError("places no longer follow the tokens' order: observe before evicting")
        b, packed_k, scales_k, valid = self._in_use()
        t, n = query.shape[0], self.n_tokens
        visible = torch.arange(n - t + 1, n + 1, dtype=torch.int32, device=self.device)
        weights = self.weights[:, :b * self.spec.block_tokens]
        watch = ops.status_watch(self.device)
        watch.poll("DeviceKVCache.observe (an earlier call)")
        _, lse = ops.attention_weights(self._rotated(query), packed_k, scales_k, valid,
                                       self.spec.bits, self.spec.group_size, self._scale(sm_scale),
                                       visible=visible, previous=weights, out=weights)
        watch.arm("DeviceKVCache.observe")
        return lse

    def evict(self, keep: int, sink: int = 0, recent: int = 0, shared: bool = False) -> None:
        """Keeps ``keep`` tokens per KV head (or the same for all, ``shared``): the first ``sink``
        positions, the ``recent`` latest, and those of the largest accumulated weight (ops.evict).
        A cache that holds no more than ``keep`` tokens is left as it is. Once the heads have chosen
        for themselves, a shared choice has no meaning any more and is refused. A failure of an earlier
        call that is known by now is raised before anything moves; ``check()`` first waits for all."""
        self._not_captured("evict")
        if keep < 1 or sink < 0 or recent < 0:
            raise ValueError("keep must be positive, sink and recent non-negative")
        if shared and self._own_choices:
            raise ValueError("the KV heads already keep different tokens")
        if self.n_tokens <= keep:
            return
        b = self.used_blocks
        ops.status_watch(self.device).poll("DeviceKVCache.evict (an earlier call)")
        if len(self._stats) == 1:
            self._stats.append(torch.empty_like(self._stats[0]))
            self._evicted = self._parts(self._stats[1])
        ops.evict(
            self.weights, self.positions, self.n_tokens, keep, self.packed_k[:b], self.packed_v[:b],
            self.scales_k[:b], self.scales_v[:b], self.valid_tokens[:b], sink=sink, recent=recent,
            next_position=self.next_position, shared=shared, out=self._evicted)
        self._stats[0].copy_(self._stats[1])  # in place: a captured decode adds to these buffers
        self.n_tokens = keep
        self._own_choices |= not shared

    def check(self) -> None:
        """Waits for this device's current stream and raises ops.DeviceFailure if any call on it flagged
        a failure."""
        watch = ops.status_watch(self.device)
        watch.arm("DeviceKVCache")  # behind all calls, those that arm no read of their own included
        watch.check("DeviceKVCache")
