"""The operators of a serving step beside the compressed projections
(include/hxq_serving.h): step plans, the 8-bit KV cache and attention over
it, and low-rank adapters of many requests.

    plan = kv_plan(new, cached, table, free, block_tokens, n_slots)
    cache = KvCache.allocate(n_blocks, n_heads, head_dim)
    cache.append(k, v, plan.slots)
    o = cache.attention(q, plan.starts, plan.lens, table, max_new=1)

    lp = lora_plan(plan.starts, adapter_ids, n_adapters, n_tokens)
    y = LoraAdapters(a, b, scales).add(y, x, lp)

The calls are made by hxq_b200/_serving.so (csrc/torch_serving.cpp).  Each
runs on the current CUDA stream of its tensors' device, takes its
outputs and workspace from PyTorch's allocator, and can be captured in a CUDA
graph.  Lengths, tables, slots and adapter numbers are int32 CUDA tensors and
are not read on the host; `status`, an int32 CUDA tensor of one element, takes
the HXQ_SERVING_* bits of what the device found out of range (see `problems`).
There is no CPU implementation, and no gradient: with grad mode on, tensors
that require one are refused.
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple

import torch

from . import lib

try:
    from . import _serving
except ImportError as e:
    raise RuntimeError("hxq_b200/_serving.so not built (run `make -C hxq-native_b200`)") from e

_serving.bind({name: C.cast(getattr(lib(), name), C.c_void_p).value for name in (
    "hxq_cuda_kv_plan", "hxq_cuda_kv_append", "hxq_cuda_kv_read", "hxq_cuda_kv_attention_workspace", "hxq_cuda_kv_attention",
    "hxq_lora_tiles", "hxq_cuda_lora_plan", "hxq_cuda_lora_workspace", "hxq_cuda_lora", "hxq_error_string")})

_PROBLEMS = {1: "the free list ran out of blocks", 2: "a block number or slot outside the cache, or a table too narrow",
             4: "a negative length, or starts outside the rows", 8: "more tokens than slots",
             16: "repeated or descending slots within a block", 32: "an adapter number out of range",
             64: "a pipeline wait ran out"}


def problems(status: torch.Tensor) -> list[str]:
    """What a status word says (reads it on the host, so it waits)."""
    word = int(status.item())
    return [text for bit, text in _PROBLEMS.items() if word & bit]


class KvPlan(NamedTuple):
    starts: torch.Tensor      # [B + 1] first row of each request
    lens: torch.Tensor        # [B] keys after this step
    slots: torch.Tensor       # [n_slots] where each row's key and value go, -1 behind the last
    positions: torch.Tensor   # [n_slots]
    taken: torch.Tensor       # [1] blocks taken from the free list


def kv_plan(new: torch.Tensor, cached: torch.Tensor, table: torch.Tensor, free: torch.Tensor, block_tokens: int,
            n_slots: int, status: torch.Tensor | None = None) -> KvPlan:
    """Maps of a step in which request b brings new[b] tokens to cached[b].
    Blocks the step begins are taken from `free` in request order and entered
    in `table` [B, width] (in place); n_slots rows of slots and positions are
    made (hxq_cuda_kv_plan)."""
    return KvPlan(*_serving.kv_plan(new, cached, table, free, block_tokens, n_slots, status))


class KvCache:
    """An 8-bit KV cache: codes [n_blocks, n_heads, block_tokens, head_dim]
    (torch.int8 or torch.float8_e4m3fn) and fp32 scales [n_blocks, n_heads]
    for keys and for values.  The tensors are the caller's and are used in
    place, at whatever memory they have when a call is made; the cache is of
    these tensors for good (k, v, k_scales and v_scales cannot be assigned)."""

    k = property(lambda self: self._tensors[0])
    v = property(lambda self: self._tensors[1])
    k_scales = property(lambda self: self._tensors[2])
    v_scales = property(lambda self: self._tensors[3])

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scales: torch.Tensor, v_scales: torch.Tensor):
        self._cache = _serving.Cache(k, v, k_scales, v_scales)
        self.device = k.device
        self.n_blocks, self.n_heads, self.block_tokens, self.head_dim = k.shape
        self._tensors = (k, v, k_scales, v_scales)

    @classmethod
    def allocate(cls, n_blocks: int, n_heads: int, head_dim: int, block_tokens: int = 16, dtype: torch.dtype = torch.int8,
                 device="cuda") -> "KvCache":
        """A cache of zeros."""
        shape = (n_blocks, n_heads, block_tokens, head_dim)
        k, v = (torch.zeros(shape, dtype=torch.int8, device=device).view(dtype) for _ in range(2))
        ks, vs = (torch.zeros(shape[:2], dtype=torch.float32, device=device) for _ in range(2))
        return cls(k, v, ks, vs)

    def append(self, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, status: torch.Tensor | None = None) -> None:
        """Quantise the rows of k and v [tokens, n_heads, head_dim] into their
        slots; negative slots are skipped (hxq_cuda_kv_append: a block's scale
        grows with its largest value, and its codes are rounded again then)."""
        self._cache.append(k, v, slots, status)

    def read(self, slots: torch.Tensor, dtype: torch.dtype = torch.bfloat16,
             status: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """The values at the slots, [n, n_heads, head_dim] of k and of v;
        zeros at negative slots."""
        return self._cache.read(slots, dtype, status)

    def attention(self, q: torch.Tensor, starts: torch.Tensor, lens: torch.Tensor, table: torch.Tensor, max_new: int,
                  scale: float | None = None, window: int = 0, causal: bool = True, out: torch.Tensor | None = None,
                  lse: torch.Tensor | None = None, status: torch.Tensor | None = None) -> torch.Tensor:
        """softmax(scale q K^T) V for rows starts[b] .. starts[b + 1] of
        q [rows, heads, head_dim] (bf16 or f16), the last tokens of request b,
        over its lens[b] keys in blocks table[b] (hxq_cuda_kv_attention).
        scale: head_dim ** -0.5 by default; window: how many keys back a row
        sees (0: all); max_new: the most rows of a request.  `lse` [rows,
        heads] fp32 takes the log of the softmax sums.  `out` may be q.  Rows
        outside every request are not written."""
        return self._cache.attention(q, starts, lens, table, max_new, scale, window, causal, out, lse, status)


class LoraPlan(NamedTuple):
    buf: torch.Tensor      # tiles, then the order
    n_tiles: int
    n_tokens: int
    n_requests: int
    n_adapters: int

    @property
    def tiles(self) -> torch.Tensor:
        """[n_tiles, 4]: adapter (-1: none), first place in order, tokens, 0."""
        return self.buf[:4 * self.n_tiles].view(-1, 4)

    @property
    def order(self) -> torch.Tensor:
        """[n_tokens] token rows sorted by adapter."""
        return self.buf[4 * self.n_tiles:]


def lora_plan(starts: torch.Tensor, adapters: torch.Tensor, n_adapters: int, n_tokens: int,
              status: torch.Tensor | None = None) -> LoraPlan:
    """Sorts the n_tokens rows of a step by the adapter of their request
    (negative: none), once for every projection of the step."""
    buf, n_tiles = _serving.lora_plan(starts, adapters, n_adapters, n_tokens, status)
    return LoraPlan(buf, n_tiles, n_tokens, adapters.numel(), n_adapters)


class LoraAdapters:
    """Low-rank adapters of one projection: a [n_adapters, rank, in_features]
    and b [n_adapters, out_features, rank] in bf16, scales [n_adapters] fp32.
    Smaller ranks are padded with zeros.  The tensors are the caller's, as a
    KvCache's are."""

    a = property(lambda self: self._tensors[0])
    b = property(lambda self: self._tensors[1])
    scales = property(lambda self: self._tensors[2])

    def __init__(self, a: torch.Tensor, b: torch.Tensor, scales: torch.Tensor):
        self._adapters = _serving.Adapters(a, b, scales)
        self.device = a.device
        self.n_adapters, self.rank, self.in_features = a.shape
        self.out_features = b.shape[1]
        self._tensors = (a, b, scales)

    def add(self, y: torch.Tensor, x: torch.Tensor, plan: LoraPlan, out: torch.Tensor | None = None) -> torch.Tensor:
        """y + scale (x A^T) B^T of each token's adapter: x [tokens,
        in_features] bf16, y [tokens, out_features] fp32 (the shared
        projection's output); out may be y.  Rows that the plan's requests do
        not cover are not written."""
        return self._adapters.add(y, x, plan.buf, plan.n_tiles, plan.n_tokens, plan.n_requests, plan.n_adapters, out)
