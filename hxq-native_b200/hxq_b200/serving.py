"""The operators of a serving step beside the compressed projections
(include/hxq_serving.h): step plans, the 8-bit KV cache and attention over
it, and low-rank adapters of many requests.

    plan = kv_plan(new, cached, table, free, block_tokens, n_slots)
    cache = KvCache.allocate(n_blocks, n_heads, head_dim)
    cache.append(k, v, plan.slots)
    o = cache.attention(q, plan.starts, plan.lens, table, max_new=1)

    lp = lora_plan(plan.starts, adapter_ids, n_adapters, n_tokens)
    y = LoraAdapters(a, b, scales).add(y, x, lp)

Every call runs on the current CUDA stream of its tensors' device, takes its
outputs and workspace from PyTorch's allocator, and can be captured in a CUDA
graph.  Lengths, tables, slots and adapter numbers are int32 CUDA tensors and
are not read on the host; `status`, an int32 CUDA tensor of one element, takes
the HXQ_SERVING_* bits of what the device found out of range (see `problems`).
There is no CPU implementation.
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple

import torch

from . import (HXQ_ELEM_BF16, HXQ_ELEM_F16, HXQ_ELEM_F32, HXQ_KV_E4M3, HXQ_KV_INT8, KvAttention, KvCacheDesc, LoraDesc,
               check, lib)

_ELEM = {torch.float32: HXQ_ELEM_F32, torch.bfloat16: HXQ_ELEM_BF16, torch.float16: HXQ_ELEM_F16}
_FORMAT = {torch.int8: HXQ_KV_INT8, torch.float8_e4m3fn: HXQ_KV_E4M3}

_PROBLEMS = {1: "the free list ran out of blocks", 2: "a block number or slot outside the cache, or a table too narrow",
             4: "a negative length, or starts outside the rows", 8: "more tokens than slots",
             16: "repeated or descending slots within a block", 32: "an adapter number out of range",
             64: "a pipeline wait ran out"}


def problems(status: torch.Tensor) -> list[str]:
    """What a status word says (reads it on the host, so it waits)."""
    word = int(status.item())
    return [text for bit, text in _PROBLEMS.items() if word & bit]


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _ints(t: torch.Tensor, name: str, dev: torch.device, dim: int = 1) -> None:
    if t.dtype != torch.int32 or t.device != dev or t.dim() != dim or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor of {dim} dimension(s) on {dev}")


def _status(status: torch.Tensor | None, dev: torch.device):
    if status is None:
        return None
    if status.dtype not in (torch.int32, torch.uint32) or status.device != dev or status.numel() != 1:
        raise ValueError(f"status must be an int32 tensor of one element on {dev}")
    return status.data_ptr()


def _cuda(t: torch.Tensor, name: str) -> torch.device:
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    return t.device


# The current device and a device's current stream as plain numbers: the
# wrapper objects of torch.cuda cost more than a launch.
_current_device = torch._C._cuda_getDevice if hasattr(torch._C, "_cuda_getDevice") else torch.cuda.current_device
if hasattr(torch._C, "_cuda_getCurrentRawStream"):
    _stream = torch._C._cuda_getCurrentRawStream
else:
    def _stream(index: int) -> int:
        return torch.cuda.current_stream(index).cuda_stream


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
    dev = _cuda(new, "new")
    _ints(new, "new", dev)
    _ints(cached, "cached", dev)
    _ints(free, "free", dev)
    _ints(table, "table", dev, 2)
    B = new.numel()
    _need(cached.numel() == B and table.shape[0] == B, "new, cached and table must have one entry per request")
    _need(0 < block_tokens <= 65536 and 0 <= n_slots < 2 ** 31, "block_tokens or n_slots out of range")
    if dev.index != _current_device():
        with torch.cuda.device(dev):
            return kv_plan(new, cached, table, free, block_tokens, n_slots, status)
    buf = torch.empty(2 * B + 2 + 2 * n_slots, dtype=torch.int32, device=dev)
    at = buf.data_ptr()
    err = lib().hxq_cuda_kv_plan(new.data_ptr(), cached.data_ptr(), B, table.data_ptr(), table.shape[1], block_tokens,
                                 free.data_ptr(), free.numel(), at, at + 4 * (B + 1), at + 4 * (2 * B + 2),
                                 at + 4 * (2 * B + 2 + n_slots), n_slots, at + 4 * (2 * B + 1), _status(status, dev),
                                 _stream(dev.index))
    if err:
        check(err, "hxq_cuda_kv_plan")
    starts, lens, taken, slots, positions = torch.split_with_sizes(buf, (B + 1, B, 1, n_slots, n_slots))
    return KvPlan(starts, lens, slots, positions, taken)


class KvCache:
    """An 8-bit KV cache: codes [n_blocks, n_heads, block_tokens, head_dim]
    (torch.int8 or torch.float8_e4m3fn) and fp32 scales [n_blocks, n_heads]
    for keys and for values.  The tensors are the caller's and are used in
    place."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scales: torch.Tensor, v_scales: torch.Tensor):
        self.device = _cuda(k, "k")
        _need(k.dtype in _FORMAT and v.dtype == k.dtype, "codes must be torch.int8 or torch.float8_e4m3fn")
        _need(k.dim() == 4 and v.shape == k.shape, "codes must be [n_blocks, n_heads, block_tokens, head_dim]")
        self.n_blocks, self.n_heads, self.block_tokens, self.head_dim = k.shape
        _need(self.head_dim in (64, 128, 256), "head_dim must be 64, 128 or 256")
        _need(self.block_tokens % 16 == 0 and 0 < self.block_tokens <= 256,
              "block_tokens must be a multiple of 16, at most 256")
        _need(self.n_blocks > 0 and self.n_heads > 0 and self.n_blocks * self.block_tokens < 2 ** 31, "cache too large or empty")
        for t in (k_scales, v_scales):
            _need(t.dtype == torch.float32 and tuple(t.shape) == (self.n_blocks, self.n_heads),
                  "scales must be fp32 [n_blocks, n_heads]")
        _need(all(t.device == self.device and t.is_contiguous() for t in (k, v, k_scales, v_scales)),
              "the cache's tensors must be contiguous and on one device")
        _need(k.data_ptr() % 16 == 0 and v.data_ptr() % 16 == 0, "codes must be 16-byte aligned")
        self.k, self.v, self.k_scales, self.v_scales = k, v, k_scales, v_scales
        self._desc = KvCacheDesc(k.data_ptr(), v.data_ptr(), k_scales.data_ptr(), v_scales.data_ptr(), self.n_blocks,
                                 self.n_heads, self.block_tokens, self.head_dim, _FORMAT[k.dtype])
        self._ref = C.byref(self._desc)

    @classmethod
    def allocate(cls, n_blocks: int, n_heads: int, head_dim: int, block_tokens: int = 16, dtype: torch.dtype = torch.int8,
                 device="cuda") -> "KvCache":
        """A cache of zeros."""
        shape = (n_blocks, n_heads, block_tokens, head_dim)
        k, v = (torch.zeros(shape, dtype=torch.int8, device=device).view(dtype) for _ in range(2))
        ks, vs = (torch.zeros(shape[:2], dtype=torch.float32, device=device) for _ in range(2))
        return cls(k, v, ks, vs)

    def _rows(self, t: torch.Tensor, name: str) -> torch.Tensor:
        _need(t.device == self.device and t.dtype in _ELEM and t.dim() == 3 and t.shape[1:] == (self.n_heads, self.head_dim),
              f"{name} must be [tokens, {self.n_heads}, {self.head_dim}] in fp32, bf16 or f16 on {self.device}")
        return t if t.stride(2) == 1 else t.contiguous()

    def append(self, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, status: torch.Tensor | None = None) -> None:
        """Quantise the rows of k and v [tokens, n_heads, head_dim] into their
        slots; negative slots are skipped (hxq_cuda_kv_append: a block's scale
        grows with its largest value, and its codes are rounded again then)."""
        k, v = self._rows(k, "k"), self._rows(v, "v")
        _ints(slots, "slots", self.device)
        _need(k.dtype == v.dtype and k.shape[0] == v.shape[0] == slots.numel(), "k, v and slots must go together")
        dev = self.device
        if dev.index != _current_device():
            with torch.cuda.device(dev):
                return self.append(k, v, slots, status)
        err = lib().hxq_cuda_kv_append(self._ref, k.data_ptr(), v.data_ptr(), _ELEM[k.dtype], k.stride(0), k.stride(1),
                                       v.stride(0), v.stride(1), slots.data_ptr(), slots.numel(), _status(status, dev),
                                       _stream(dev.index))
        if err:
            check(err, "hxq_cuda_kv_append")

    def read(self, slots: torch.Tensor, dtype: torch.dtype = torch.bfloat16,
             status: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """The values at the slots, [n, n_heads, head_dim] of k and of v;
        zeros at negative slots."""
        _ints(slots, "slots", self.device)
        _need(dtype in _ELEM, "dtype must be fp32, bf16 or f16")
        dev = self.device
        if dev.index != _current_device():
            with torch.cuda.device(dev):
                return self.read(slots, dtype, status)
        k, v = torch.empty((2, slots.numel(), self.n_heads, self.head_dim), dtype=dtype, device=dev).unbind()
        err = lib().hxq_cuda_kv_read(self._ref, slots.data_ptr(), slots.numel(), k.data_ptr(), v.data_ptr(), _ELEM[dtype],
                                     _status(status, dev), _stream(dev.index))
        if err:
            check(err, "hxq_cuda_kv_read")
        return k, v

    def attention(self, q: torch.Tensor, starts: torch.Tensor, lens: torch.Tensor, table: torch.Tensor, max_new: int,
                  scale: float | None = None, window: int = 0, causal: bool = True, out: torch.Tensor | None = None,
                  lse: torch.Tensor | None = None, status: torch.Tensor | None = None) -> torch.Tensor:
        """softmax(scale q K^T) V for rows starts[b] .. starts[b + 1] of
        q [rows, heads, head_dim] (bf16 or f16), the last tokens of request b,
        over its lens[b] keys in blocks table[b] (hxq_cuda_kv_attention).
        scale: head_dim ** -0.5 by default; window: how many keys back a row
        sees (0: all); max_new: the most rows of a request.  `lse` [rows,
        heads] fp32 takes the log of the softmax sums.  Rows outside every
        request are not written."""
        dev = self.device
        _need(q.device == dev and q.dtype in (torch.bfloat16, torch.float16) and q.dim() == 3
              and q.shape[2] == self.head_dim and q.shape[1] > 0 and q.shape[1] % self.n_heads == 0,
              f"q must be [rows, a multiple of {self.n_heads}, {self.head_dim}] in bf16 or f16 on {dev}")
        if q.stride(2) != 1 or (q.stride(0) | q.stride(1)) % 8 or q.data_ptr() % 16:
            q = q.clone(memory_format=torch.contiguous_format)
        _ints(starts, "starts", dev)
        _ints(lens, "lens", dev)
        _ints(table, "table", dev, 2)
        B, T = lens.numel(), q.shape[0]
        _need(starts.numel() == B + 1 and table.shape[0] == B, "starts must have one entry more than lens, table as many")
        _need(window >= 0 and (causal or not window), "a window needs causal attention")
        _need(lse is None or (lse.dtype == torch.float32 and lse.is_contiguous() and tuple(lse.shape) == tuple(q.shape[:2])
                              and lse.device == dev), "lse must be fp32 [rows, heads]")
        if dev.index != _current_device():
            with torch.cuda.device(dev):
                return self.attention(q, starts, lens, table, max_new, scale, window, causal, out, lse, status)
        if out is None:
            out = torch.empty(q.shape, dtype=q.dtype, device=dev)
        else:
            _need(out.shape == q.shape and out.dtype == q.dtype and out.device == dev and out.stride(2) == 1,
                  "out must be like q")
        p = KvAttention(q.data_ptr(), out.data_ptr(), None if lse is None else lse.data_ptr(), q.stride(0), q.stride(1),
                        out.stride(0), out.stride(1), starts.data_ptr(), lens.data_ptr(), table.data_ptr(), B, T,
                        q.shape[1], table.shape[1], max_new, window, self.head_dim ** -0.5 if scale is None else scale,
                        _ELEM[q.dtype], 1 if causal else 0)
        L, ref = lib(), C.byref(p)
        size = L.hxq_cuda_kv_attention_workspace(self._ref, ref)
        ws = torch.empty(size, dtype=torch.uint8, device=dev)
        err = L.hxq_cuda_kv_attention(self._ref, ref, ws.data_ptr(), size, _status(status, dev), _stream(dev.index))
        if err:
            check(err, "hxq_cuda_kv_attention")
        return out


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
    dev = _cuda(starts, "starts")
    _ints(starts, "starts", dev)
    _ints(adapters, "adapters", dev)
    B = adapters.numel()
    _need(starts.numel() == B + 1, "starts must have one entry more than adapters")
    _need(0 < n_adapters <= 4096 and 0 <= n_tokens < 2 ** 31, "n_adapters or n_tokens out of range")
    if dev.index != _current_device():
        with torch.cuda.device(dev):
            return lora_plan(starts, adapters, n_adapters, n_tokens, status)
    L = lib()
    n_tiles = L.hxq_lora_tiles(B, n_adapters, n_tokens)
    buf = torch.empty(4 * n_tiles + n_tokens, dtype=torch.int32, device=dev)
    at = buf.data_ptr()
    err = L.hxq_cuda_lora_plan(starts.data_ptr(), adapters.data_ptr(), B, n_adapters, n_tokens, at + 16 * n_tiles, at,
                               _status(status, dev), _stream(dev.index))
    if err:
        check(err, "hxq_cuda_lora_plan")
    return LoraPlan(buf, n_tiles, n_tokens, B, n_adapters)


class LoraAdapters:
    """Low-rank adapters of one projection: a [n_adapters, rank, in_features]
    and b [n_adapters, out_features, rank] in bf16, scales [n_adapters] fp32.
    Smaller ranks are padded with zeros."""

    def __init__(self, a: torch.Tensor, b: torch.Tensor, scales: torch.Tensor):
        self.device = _cuda(a, "a")
        _need(a.dtype == b.dtype == torch.bfloat16 and a.dim() == b.dim() == 3, "a and b must be bf16 with three dimensions")
        self.n_adapters, self.rank, self.in_features = a.shape
        self.out_features = b.shape[1]
        _need(tuple(b.shape) == (self.n_adapters, self.out_features, self.rank), "b must be [n_adapters, out_features, rank]")
        _need(self.rank % 8 == 0 and 0 < self.rank <= 128, "rank must be a multiple of 8, at most 128")
        _need(self.in_features % 8 == 0 and self.in_features > 0 and self.out_features > 0, "in_features must be a multiple of 8")
        _need(0 < self.n_adapters <= 4096, "between 1 and 4096 adapters")
        _need(scales.dtype == torch.float32 and tuple(scales.shape) == (self.n_adapters,), "scales must be fp32 [n_adapters]")
        _need(all(t.device == self.device and t.is_contiguous() for t in (a, b, scales)),
              "the adapters' tensors must be contiguous and on one device")
        _need(a.data_ptr() % 16 == 0 and b.data_ptr() % 16 == 0, "a and b must be 16-byte aligned")
        self.a, self.b, self.scales = a, b, scales
        self._desc = LoraDesc(a.data_ptr(), b.data_ptr(), scales.data_ptr(), self.n_adapters, self.rank, self.in_features,
                              self.out_features)
        self._ref = C.byref(self._desc)

    def add(self, y: torch.Tensor, x: torch.Tensor, plan: LoraPlan, out: torch.Tensor | None = None) -> torch.Tensor:
        """y + scale (x A^T) B^T of each token's adapter: x [tokens,
        in_features] bf16, y [tokens, out_features] fp32 (the shared
        projection's output); out may be y.  Rows that the plan's requests do
        not cover are not written."""
        dev = self.device
        _need(x.device == dev and x.dtype == torch.bfloat16 and x.dim() == 2 and x.shape[1] == self.in_features,
              f"x must be bf16 [tokens, {self.in_features}] on {dev}")
        T = x.shape[0]
        _need(y.device == dev and y.dtype == torch.float32 and tuple(y.shape) == (T, self.out_features),
              f"y must be fp32 [tokens, {self.out_features}] on {dev}")
        _need(plan.n_adapters == self.n_adapters and plan.n_tokens == T and plan.buf.device == dev,
              "the plan was made for other adapters or tokens")
        if x.stride(1) != 1 or x.stride(0) % 8 or x.data_ptr() % 16:
            x = x.clone(memory_format=torch.contiguous_format)
        if y.stride(1) != 1:
            _need(out is not y, "y must have consecutive elements to be written in place")
            y = y.contiguous()
        if dev.index != _current_device():
            with torch.cuda.device(dev):
                return self.add(y, x, plan, out)
        if out is None:
            out = torch.empty((T, self.out_features), dtype=torch.float32, device=dev)
        else:
            _need(out.device == dev and out.dtype == torch.float32 and out.shape == y.shape and out.stride(1) == 1,
                  "out must be like y")
        L = lib()
        size = L.hxq_cuda_lora_workspace(self._ref, plan.n_requests, T)
        ws, at = torch.empty(size, dtype=torch.uint8, device=dev), plan.buf.data_ptr()
        err = L.hxq_cuda_lora(self._ref, x.data_ptr(), x.stride(0), y.data_ptr(), y.stride(0), out.data_ptr(), out.stride(0),
                              plan.n_requests, T, at + 16 * plan.n_tiles, at, ws.data_ptr(), size, _stream(dev.index))
        if err:
            check(err, "hxq_cuda_lora")
        return out
