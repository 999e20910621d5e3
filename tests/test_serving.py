"""The serving operators (include/hxq_serving.h, hxq_b200.serving): step plans,
the 8-bit KV cache, attention over it and low-rank adapters, each against a
plain implementation in 64 bits, at the sizes and masks where it can go wrong;
refusals; a step of all of them together."""
import ctypes as C
import math

import pytest

FAKE = 0x7f0000000000   # a pointer that no refused call may touch


# -- refusals (no GPU) ---------------------------------------------------------

def _cache(H, **kw):
    d = dict(k=FAKE, v=FAKE, k_scales=FAKE, v_scales=FAKE, n_blocks=8, n_heads=2, block_tokens=16, head_dim=64, format=0)
    d.update(kw)
    return H.KvCacheDesc(**d)


@pytest.mark.parametrize("bad,code", [
    (dict(k=None), 1), (dict(v_scales=None), 1), (dict(head_dim=96), 3), (dict(block_tokens=24), 3), (dict(block_tokens=0), 3),
    (dict(block_tokens=272), 3), (dict(n_blocks=0), 34), (dict(n_heads=0), 34), (dict(format=2), 34), (dict(k=FAKE + 8), 34),
    (dict(n_blocks=1 << 28), 34)])
def test_cache_refusals(H, L, bad, code):
    c = _cache(H, **bad)
    assert L.hxq_cuda_kv_append(C.byref(c), FAKE, FAKE, 1, 128, 64, 128, 64, FAKE, 4, None, None) == code
    assert L.hxq_cuda_kv_read(C.byref(c), FAKE, 4, FAKE, FAKE, 1, None, None) == code
    a = H.KvAttention(q=FAKE, out=FAKE, starts=FAKE, lens=FAKE, table=FAKE, n_requests=1, n_rows=1, n_heads=2, table_width=1,
                      max_new=1, scale=1.0, elem=1, causal=1)
    assert L.hxq_cuda_kv_attention(C.byref(c), C.byref(a), FAKE, 1 << 40, None, None) == code
    assert L.hxq_cuda_kv_attention_workspace(C.byref(c), C.byref(a)) == 0


def test_append_and_read_refusals(H, L):
    c = C.byref(_cache(H))
    assert L.hxq_cuda_kv_append(None, FAKE, FAKE, 1, 128, 64, 128, 64, FAKE, 4, None, None) == 1
    assert L.hxq_cuda_kv_append(c, None, FAKE, 1, 128, 64, 128, 64, FAKE, 4, None, None) == 1
    assert L.hxq_cuda_kv_append(c, FAKE, FAKE, 1, 128, 64, 128, 64, None, 4, None, None) == 1
    assert L.hxq_cuda_kv_append(c, FAKE, FAKE, 3, 128, 64, 128, 64, FAKE, 4, None, None) == 34
    assert L.hxq_cuda_kv_append(c, FAKE + 1, FAKE, 1, 128, 64, 128, 64, FAKE, 4, None, None) == 34
    assert L.hxq_cuda_kv_append(c, None, None, 1, 128, 64, 128, 64, None, 0, None, None) == 0
    assert L.hxq_cuda_kv_read(c, FAKE, 4, None, None, 1, None, None) == 1
    assert L.hxq_cuda_kv_read(c, FAKE, 4, FAKE, FAKE, 7, None, None) == 34
    assert L.hxq_cuda_kv_read(c, None, 0, None, None, 1, None, None) == 0


@pytest.mark.parametrize("bad,code", [
    (dict(elem=0), 34), (dict(n_heads=3), 3), (dict(n_heads=0), 3), (dict(window=4, causal=0), 34), (dict(scale=-1.0), 34),
    (dict(scale=math.inf), 34), (dict(scale=math.nan), 34), (dict(n_requests=8193), 34), (dict(table_width=1 << 28), 34),
    (dict(q=None), 1), (dict(out=None), 1), (dict(starts=None), 1), (dict(lens=None), 1), (dict(table=None), 1),
    (dict(q=FAKE + 8), 34), (dict(q_stride_t=100), 34)])
def test_attention_refusals(H, L, bad, code):
    d = dict(q=FAKE, out=FAKE, starts=FAKE, lens=FAKE, table=FAKE, n_requests=1, n_rows=1, n_heads=4, table_width=1, max_new=1,
             scale=1.0, elem=1, causal=1, q_stride_t=256, q_stride_h=64, out_stride_t=256, out_stride_h=64)
    d.update(bad)
    a = H.KvAttention(**d)
    assert L.hxq_cuda_kv_attention(C.byref(_cache(H)), C.byref(a), FAKE, 1 << 40, None, None) == code
    a = H.KvAttention(**{**d, **dict(bad), "n_rows": 0}) if code == 1 else a
    if code == 1:
        assert L.hxq_cuda_kv_attention(C.byref(_cache(H)), C.byref(a), FAKE, 1 << 40, None, None) == 0


def test_attention_workspace_refusals(H, L):
    a = H.KvAttention(q=FAKE, out=FAKE, starts=FAKE, lens=FAKE, table=FAKE, n_requests=1, n_rows=1, n_heads=4, table_width=1,
                      max_new=1, scale=1.0, elem=1, causal=1, q_stride_t=256, q_stride_h=64)
    c = C.byref(_cache(H))
    size = L.hxq_cuda_kv_attention_workspace(c, C.byref(a))
    assert size > 0
    assert L.hxq_cuda_kv_attention(c, C.byref(a), FAKE, size - 1, None, None) == 34
    assert L.hxq_cuda_kv_attention(c, C.byref(a), None, size, None, None) == 1
    assert L.hxq_cuda_kv_attention(c, C.byref(a), FAKE + 4, size, None, None) == 34
    assert L.hxq_cuda_kv_attention(c, None, FAKE, size, None, None) == 1


def test_plan_refusals(H, L):
    def call(**kw):
        d = dict(new=FAKE, cached=FAKE, B=2, table=FAKE, width=4, P=16, free=FAKE, n_free=4, starts=FAKE, lens=FAKE, slots=FAKE,
                 pos=FAKE, n=8, taken=FAKE, status=None, stream=None)
        d.update(kw)
        return L.hxq_cuda_kv_plan(*d.values())
    for name in ("new", "cached", "table", "free", "starts", "lens", "slots", "pos", "taken"):
        assert call(**{name: None}) == 1, name
    assert call(P=0) == 34 and call(P=65537) == 34 and call(B=8193) == 34 and call(n=1 << 31) == 34


def test_lora_refusals(H, L):
    def call(l=None, x=FAKE, ldx=64, y=FAKE, out=FAKE, B=2, T=4, order=FAKE, tiles=FAKE, ws=FAKE, size=1 << 40, **kw):
        d = dict(a=FAKE, b=FAKE, scales=FAKE, n_adapters=2, rank=16, in_features=64, out_features=48)
        d.update(kw)
        return L.hxq_cuda_lora(C.byref(H.LoraDesc(**d)), x, ldx, y, 48, out, 48, B, T, order, tiles, ws, size, None)
    for kw in (dict(a=None), dict(b=None), dict(scales=None), dict(x=None), dict(y=None), dict(out=None), dict(order=None),
               dict(tiles=None), dict(ws=None)):
        assert call(**kw) == 1, kw
    for kw in (dict(rank=0), dict(rank=12), dict(rank=136), dict(in_features=60), dict(out_features=0)):
        assert call(**kw) == 3, kw
    for kw in (dict(n_adapters=0), dict(n_adapters=4097), dict(x=FAKE + 8), dict(ldx=63), dict(size=0), dict(B=8193), dict(tiles=FAKE + 4)):
        assert call(**kw) == 34, kw
    assert call(T=0) == 0 and call(B=0) == 0
    assert L.hxq_cuda_lora_plan(None, FAKE, 2, 2, 4, FAKE, FAKE, None, None) == 1
    assert L.hxq_cuda_lora_plan(FAKE, FAKE, 2, 0, 4, FAKE, FAKE, None, None) == 34
    assert L.hxq_cuda_lora_plan(FAKE, FAKE, 8193, 2, 4, FAKE, FAKE, None, None) == 34
    # tiles: every group may end in a partly filled one, and none is empty
    assert L.hxq_lora_tiles(1, 4, 1) == 1 and L.hxq_lora_tiles(3, 8, 200) == 6 and L.hxq_lora_tiles(50, 8, 2000) == 40


def test_python_refusals():
    import torch

    from hxq_b200 import serving as S
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError):
        S.kv_plan(i, i, i.view(2, 1), i, 16, 4)
    with pytest.raises(ValueError):
        S.KvCache.allocate(4, 2, 64, device="cpu")
    with pytest.raises(ValueError):
        S.lora_plan(i, i, 2, 4)
    with pytest.raises(ValueError):
        S.LoraAdapters(torch.zeros(1, 8, 8, dtype=torch.bfloat16), torch.zeros(1, 8, 8, dtype=torch.bfloat16), torch.ones(1))


# -- plan ------------------------------------------------------------------------

def _plan_ref(new, cached, table, free, P, n_slots):
    table, starts, slots, pos, used = [list(r) for r in table], [0], [], [], 0
    for b, (n, c) in enumerate(zip(new, cached)):
        for j in range(-(-c // P), -(-(c + n) // P)):
            e = free[used] if used < len(free) else -1
            used += 1
            if j < len(table[b]):
                table[b][j] = e
        for p in range(c, c + n):
            blk = table[b][p // P] if p // P < len(table[b]) else -1
            slots.append(blk * P + p % P if blk >= 0 else -1)
            pos.append(p)
        starts.append(starts[-1] + n)
    pad = n_slots - len(slots)
    return (starts, [c + n for n, c in zip(new, cached)], table, (slots + [-1] * max(pad, 0))[:n_slots],
            (pos + [-1] * max(pad, 0))[:n_slots], min(used, len(free)))


@pytest.mark.gpu
@pytest.mark.parametrize("B,most,held,P,free,pad,width", [
    (1, 1, 0, 16, 9, 0, 8), (3, 1, 40, 16, 9, 5, 8), (64, 1, 500, 16, 64, 0, 40), (7, 90, 100, 32, 60, 3, 8), (5, 60, 70, 16, 4, 0, 12),
    (4, 100, 60, 16, 50, 2, 3), (700, 20, 50, 16, 2000, 11, 8), (1300, 3, 5, 128, 1300, 0, 1), (2, 5000, 1, 64, 400, 0, 90),
    (6, 50, 20, 16, 40, -30, 8), (8192, 2, 3, 16, 9000, 1, 1)])
def test_plan(cuda, B, most, held, P, free, pad, width):
    torch = cuda
    from hxq_b200 import serving as S
    g = torch.Generator().manual_seed(B * 7 + most)
    new = torch.randint(0, most + 1, (B,), generator=g, dtype=torch.int32)
    cached = torch.randint(0, held + 1, (B,), generator=g, dtype=torch.int32)
    if B > 2:
        new[1] = 0
        cached[2] = P if held >= P else 0   # a full block: the next token begins another
    table = torch.randint(1000, 5000, (B, width), generator=g, dtype=torch.int32)
    fl = torch.randperm(1000 + free, generator=g)[:free].to(torch.int32)
    n_slots = max(int(new.sum()) + pad, 0)
    want = _plan_ref(new.tolist(), cached.tolist(), table.tolist(), fl.tolist(), P, n_slots)
    t, status = table.cuda(), torch.zeros(1, dtype=torch.int32, device="cuda")
    p = S.kv_plan(new.cuda(), cached.cuda(), t, fl.cuda(), P, n_slots, status=status)
    assert p.starts.tolist() == want[0] and p.lens.tolist() == want[1]
    assert t.tolist() == want[2]
    assert p.slots.tolist() == want[3] and p.positions.tolist() == want[4] and p.taken.tolist() == [want[5]]
    need = sum(-(-(c + n) // P) - -(-c // P) for n, c in zip(new.tolist(), cached.tolist()))
    narrow = any(-(-(c + n) // P) > width for n, c in zip(new.tolist(), cached.tolist()) if n)
    assert int(status) == (1 if need > free else 0) | (2 if narrow else 0) | (8 if pad < 0 else 0), S.problems(status)


@pytest.mark.gpu
def test_plan_bad_lengths_and_empty(cuda):
    torch = cuda
    from hxq_b200 import serving as S
    i = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    status = i(0)
    p = S.kv_plan(i(2, -3, 1), i(-1, 4, 15), torch.full((3, 2), 7, dtype=torch.int32, device="cuda"), i(9, 8), 16, 4, status=status)
    assert p.starts.tolist() == [0, 2, 2, 3] and p.slots.tolist() == [144, 145, 7 * 16 + 15, -1] and int(status) == 4
    p = S.kv_plan(i(), i(), torch.zeros((0, 2), dtype=torch.int32, device="cuda"), i(), 16, 3)
    assert p.starts.tolist() == [0] and p.slots.tolist() == [-1] * 3 and p.taken.tolist() == [0]


# -- cache -------------------------------------------------------------------------

QMAX = {"int8": 127.0, "e4m3": 448.0}


def _types(torch):
    return {"int8": torch.int8, "e4m3": torch.float8_e4m3fn, "bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _append_ref(torch, codes, scales, x, slots, P, fmt):
    """The rule in fp32 (every step of it one rounding), block by block."""
    q, dt = QMAX[fmt], codes.dtype
    fit = (lambda v: v.round().clamp(-q, q).to(torch.int8)) if fmt == "int8" else (lambda v: v.clamp(-q, q).to(dt))
    vals, x = codes.float(), x.float()
    by = {}
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < codes.shape[0] * P:
            by.setdefault(s // P, []).append((t, s % P))
    for blk, rows in by.items():
        ts, ps = [r[0] for r in rows], [r[1] for r in rows]
        fresh = ps[0] == 0
        old = torch.zeros_like(scales[blk]) if fresh else scales[blk].clone()
        s = torch.maximum(old, x[ts].abs().amax(-1).amax(0) / q)
        s = torch.where(s < 2.0 ** -126, torch.zeros_like(s), s)
        for h in range(s.numel()):
            inv = 1.0 / s[h] if s[h] > 0 else torch.tensor(0.0)
            if not fresh and s[h] > old[h]:
                keep = [p for p in range(P) if p not in ps]
                vals[blk, h, keep] = fit(vals[blk, h, keep] * (old[h] / s[h])).float()
            vals[blk, h, ps] = fit(x[ts, h] * inv).float()
        scales[blk] = s
    return vals, scales


def _filled(torch, S, n_blocks, heads, dim, P, fmt, seed):
    g = torch.Generator().manual_seed(seed)
    c = S.KvCache.allocate(n_blocks, heads, dim, P, _types(torch)[fmt])
    for t in (c.k, c.v):
        x = torch.randn(t.shape, generator=g).clamp(-3, 3) * (QMAX[fmt] / 3)
        t.view(torch.int8).copy_(x.to(t.dtype).view(torch.int8))
    for t in (c.k_scales, c.v_scales):
        t.copy_(torch.rand(t.shape, generator=g) * 0.02 + 0.01)
    return c, g


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("elem,dim,heads,P,runs,layout", [
    ("bf16", 128, 2, 16, [(3, 5, 1)], "plain"), ("f16", 64, 3, 16, [(0, 0, 16), (1, 0, 9), (5, 15, 1)], "plain"),
    ("f32", 256, 1, 32, [(2, 0, 32), (3, 1, 31), (7, 30, 2)], "plain"), ("bf16", 64, 5, 256, [(0, 0, 256), (1, 100, 77)], "plain"),
    ("bf16", 128, 4, 16, [(i, (7 * i) % 16, 1) for i in range(40)], "heads first"),
    ("f16", 128, 2, 64, [(1, 3, 50), (0, 0, 64), (2, 0, 1)], "odd"), ("f32", 64, 1, 16, [(4, 2, 3)], "odd"),
    ("bf16", 128, 8, 32, [(i, 0, 32) for i in range(50)] + [(50, 0, 7)], "plain")])
def test_append_and_read(cuda, fmt, elem, dim, heads, P, runs, layout):
    torch = cuda
    from hxq_b200 import serving as S
    dt = _types(torch)
    n_blocks = max(r[0] for r in runs) + 3
    c, g = _filled(torch, S, n_blocks, heads, dim, P, fmt, 5)
    slots = [b * P + p + i for b, p, n in runs for i in range(n)]
    slots = [-1] + slots + [-1, n_blocks * P + 3]
    T = len(slots)
    x = torch.randn((2, T, heads, dim), generator=g) * torch.exp(torch.randn((2, T, 1, 1), generator=g))
    x[0, 1, 0] = 0
    want = [_append_ref(torch, t.cpu(), s.cpu(), xx.to(dt[elem]), torch.tensor(slots), P, fmt)
            for t, s, xx in ((c.k, c.k_scales, x[0]), (c.v, c.v_scales, x[1]))]
    xd = x.to(dt[elem]).cuda()
    if layout == "heads first":
        xd = xd.transpose(1, 2).contiguous().transpose(1, 2)
    elif layout == "odd":   # rows that begin anywhere
        wide = torch.empty((2, T, heads, dim + 3), dtype=dt[elem], device="cuda")
        wide[..., 1:dim + 1] = xd
        xd = wide[..., 1:dim + 1]
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    sl = torch.tensor(slots, dtype=torch.int32, device="cuda")
    c.append(xd[0], xd[1], sl, status=status)
    assert int(status) == 2
    for codes, scales, (vals, s) in ((c.k, c.k_scales, want[0]), (c.v, c.v_scales, want[1])):
        assert torch.equal(scales.cpu(), s)
        assert torch.equal(codes.float().cpu(), vals)
    # again: nothing grows, nothing moves (blocks begun anew included)
    before = [t.clone() for t in (c.k.view(torch.int8), c.v.view(torch.int8), c.k_scales, c.v_scales)]
    c.append(xd[0], xd[1], sl)
    assert all(torch.equal(a, b) for a, b in zip(before, (c.k.view(torch.int8), c.v.view(torch.int8), c.k_scales, c.v_scales)))
    for out in ("f32", "bf16", "f16"):
        status.zero_()
        for got, (vals, s), xx in zip(c.read(sl, dt[out], status=status), want, x):
            ok = torch.tensor([0 <= v < n_blocks * P for v in slots])
            at = torch.tensor(slots).clamp(0, n_blocks * P - 1)
            ref = (vals[at // P, :, at % P] * s[at // P][..., None]).to(dt[out])
            ref[~ok] = 0
            assert torch.equal(got.cpu(), ref)
            if out == "f32":   # within half a step of what was written
                xe, sc = xx.to(dt[elem]).double()[ok], s[at // P].double()[ok][..., None]
                half = sc * 0.5 if fmt == "int8" else torch.maximum(xe.abs() * 2.0 ** -4, sc * 2.0 ** -10)
                # the code is of x * (1 / scale): three roundings away from x / scale
                assert bool(((got.cpu().double()[ok] - xe).abs() <= half * (1 + 2.0 ** -14) + 448 * sc * 2.0 ** -22).all())
        assert int(status) == 2


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_append_extremes(cuda, fmt):
    torch = cuda
    from hxq_b200 import serving as S
    c = S.KvCache.allocate(6, 2, 64, 16, _types(torch)[fmt])
    x = torch.randn(6, 2, 64).cuda()
    x[0] = 0                # a block of zeros
    x[1] *= 1e-42           # below every scale
    x[2, 0, 3] = math.inf
    x[3, 0, 5] = -math.nan
    x[4] *= 1e37            # near the top of fp32
    slots = torch.tensor([b * 16 for b in range(6)], dtype=torch.int32, device="cuda")
    c.append(x, x, slots)
    k, v = c.read(slots, torch.float32)
    assert bool((k[:2] == 0).all()) and bool((c.k_scales[:2] == 0).all())
    assert bool(k[2, 0].isnan().all()) and bool(k[3, 0].isnan().all()) and bool(v[2, 0].isnan().all())
    assert bool(k[2, 1].isfinite().all()) and bool(k[3, 1].isfinite().all()) and bool(k[4:].isfinite().all())
    assert bool((c.k.float()[:, :, 0].isfinite()).all())
    # the block's first slot begins it anew
    c.append(torch.ones_like(x), torch.ones_like(x), slots)
    k, _ = c.read(slots, torch.float32)
    assert bool(((k - 1).abs() <= 2.0 ** -22).all())


@pytest.mark.gpu
def test_append_order_is_recorded(cuda):
    torch = cuda
    from hxq_b200 import serving as S
    for slots, bits in (([3, 3], 16), ([5, 4], 16), ([4, 5], 0), ([5, 20], 0), ([20, 5], 0)):
        c = S.KvCache.allocate(4, 1, 64)
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        x = torch.randn(2, 1, 64, device="cuda")
        c.append(x, x, torch.tensor(slots, dtype=torch.int32, device="cuda"), status=status)
        assert int(status) == bits, slots
        assert bool(c.k_scales.isfinite().all())


# -- attention ---------------------------------------------------------------------

def _attention_ref(torch, c, q, starts, lens, table, scale, window, causal):
    """Outputs, lse and elementwise bounds, in 64 bits."""
    G, P, D = q.shape[1] // c.n_heads, c.block_tokens, c.head_dim
    out = torch.full(q.shape, math.nan, dtype=torch.float64, device="cuda")
    lse = torch.full(q.shape[:2], math.nan, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(out)
    tol_lse = torch.zeros_like(lse)
    top = QMAX["int8" if c.k.dtype == torch.int8 else "e4m3"]
    eps = torch.finfo(q.dtype).eps / 2
    for b, n in enumerate(lens):
        s, e = starts[b], starts[b + 1]
        m = e - s
        if m <= 0:
            continue
        if n == 0:
            out[s:e], lse[s:e] = 0, -math.inf
            continue
        pages = table[b, :-(-n // P)].long()
        pos = torch.arange(n - m, n, device="cuda")
        j = torch.arange(n, device="cuda")
        mask = torch.zeros((m, n), dtype=torch.bool, device="cuda")
        if causal:
            mask |= j[None] > pos[:, None]
            if window:
                mask |= j[None] <= pos[:, None] - window
        for h in range(c.n_heads):
            ks = c.k_scales[pages, h].double().repeat_interleave(P)[:n]
            vs = c.v_scales[pages, h].double().repeat_interleave(P)[:n]
            k = c.k[pages, h].double().reshape(-1, D)[:n] * ks[:, None]
            v = c.v[pages, h].double().reshape(-1, D)[:n] * vs[:, None]
            for g in range(G):
                qq = q[s:e, h * G + g].double()
                sc = (qq @ k.T * scale).masked_fill(mask, -math.inf)
                most = sc.amax(-1, keepdim=True)
                p = torch.exp(sc - torch.where(most.isfinite(), most, 0.0))
                total = p.sum(-1, keepdim=True)
                p = torch.where(total > 0, p / total, 0.0)
                o = p @ v
                # sums of D products in fp32 (2^-23 a step covers truncating sums), the scale and the exponent's argument
                # rounded (2^-21 of it), exp2 2^-22: a weight's relative error
                size = (qq.abs() @ k.abs().T * scale).masked_fill(mask, 0).amax(-1, keepdim=True)
                ds = size * (D + 8) * 2.0 ** -23 + (size + vs.clamp(min=2.0 ** -100).log2().abs().max()) * 2.0 ** -21 + 2.0 ** -20
                w = (p * vs).amax(-1, keepdim=True)
                # weights in f16: 2^-11 of each, 2^-25 of the largest below 2^-14 of it; sums of n terms in fp32
                live = (~mask).sum(-1, keepdim=True)
                tol[s:e, h * G + g] = (eps * o.abs() + (2.0 ** -11 + 2 * ds + (live / 16 + 64) * 2.0 ** -23) * (p @ v.abs())
                                       + w * live * top * 2.0 ** -25 + torch.finfo(q.dtype).smallest_normal * eps)
                out[s:e, h * G + g] = o
                lse[s:e, h * G + g] = (most + total.log())[:, 0]
                tol_lse[s:e, h * G + g] = (2 * ds + (live / 16 + 64) * 2.0 ** -23)[:, 0] + (most.abs() * 2.0 ** -22)[:, 0]
    return out, lse, tol, tol_lse


def _attention_case(torch, S, new, lens, heads, group, dim, P, fmt, elem, seed=3, spread=1.0):
    need = [-(-n // P) for n in lens]
    n_blocks = sum(need) + 3
    c, g = _filled(torch, S, n_blocks, heads, dim, P, fmt, seed)
    for t in (c.k_scales, c.v_scales):
        t.copy_(torch.exp(spread * torch.randn(t.shape, generator=g)) / QMAX[fmt])
    order = torch.randperm(n_blocks, generator=g).tolist()
    W = max(max(need), 1) + 1
    table = torch.full((len(lens), W), -7, dtype=torch.int32)   # entries behind a request's blocks are never used
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor([order.pop() for _ in range(n)], dtype=torch.int32)
        if n and lens[b] % P:   # what is behind the last key may be anything, NaN codes among it
            c.k.view(torch.uint8)[int(table[b, n - 1]), :, lens[b] % P:] = 0x7f
            c.v.view(torch.uint8)[int(table[b, n - 1]), :, lens[b] % P:] = 0xff
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    q = torch.randn((starts[-1], heads * group, dim), generator=g).to(_types(torch)[elem]).cuda()
    i = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    return c, q, starts, i(starts), i(lens), table.cuda()


def _check_attention(torch, S, c, q, starts, starts_d, lens_d, table, max_new, window=0, causal=True, scale=None, **kw):
    lse = torch.full(q.shape[:2], 7.0, dtype=torch.float32, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    o = c.attention(q, starts_d, lens_d, table, max_new, scale=scale, window=window, causal=causal, lse=lse, status=status, **kw)
    assert int(status) == 0, S.problems(status)
    want, wl, tol, tl = _attention_ref(torch, c, q, starts, lens_d.tolist(), table, c.head_dim ** -0.5 if scale is None else scale,
                                       window, causal)
    n = starts[-1]
    over = (o[:n].double() - want[:n]).abs() - tol[:n]
    assert bool((over <= 0).all()), (float(over.max()), float((o[:n].double() - want[:n]).abs().max()))
    fin = wl[:n].isfinite()
    assert torch.equal(fin, lse[:n].isfinite())
    assert bool(((lse[:n].double() - wl[:n])[fin].abs() <= tl[:n][fin]).all())
    again = c.attention(q, starts_d, lens_d, table, max_new, scale=scale, window=window, causal=causal, **kw)
    assert torch.equal(again[:n], o[:n])   # the same bits every time
    return o, lse


SHAPES = [
    # new, lens, heads, group, dim, block, window, causal
    ([1], [1], 1, 1, 128, 16, 0, True),
    ([1], [17], 2, 4, 64, 16, 0, True),
    ([1, 1, 1], [64, 65, 15], 2, 8, 128, 16, 0, True),
    ([1] * 5, [1000, 3, 0, 257, 16], 1, 5, 128, 32, 0, True),
    ([1, 2, 0, 3], [5, 2, 40, 3], 3, 7, 64, 64, 0, True),
    ([4, 1], [700, 900], 2, 16, 128, 128, 0, True),
    ([1, 5], [300, 90], 2, 2, 256, 16, 0, True),
    ([1, 3], [3000, 500], 1, 1, 64, 256, 100, True),
    ([2, 9], [40, 200], 2, 3, 128, 16, 1, True),
    ([33, 1, 20], [33, 70, 300], 2, 4, 128, 16, 0, True),
    ([70, 130], [70, 1000], 1, 2, 64, 32, 33, True),
    ([5, 9], [77, 20], 2, 3, 64, 16, 0, False),
    ([40], [100], 1, 3, 256, 64, 17, True),
    ([5], [3], 1, 4, 128, 16, 0, True),           # rows before position 0 see nothing
    ([1], [40000], 1, 1, 128, 64, 0, True),
    ([200, 1, 300], [200, 4000, 1300], 2, 5, 128, 16, 0, True),
]


@pytest.mark.gpu
@pytest.mark.parametrize("fmt,elem", [("int8", "bf16"), ("e4m3", "f16"), ("int8", "f16"), ("e4m3", "bf16")])
@pytest.mark.parametrize("case", range(len(SHAPES)))
def test_attention(cuda, case, fmt, elem):
    torch = cuda
    from hxq_b200 import serving as S
    new, lens, heads, group, dim, P, window, causal = SHAPES[case]
    c, q, starts, sd, ld, table = _attention_case(torch, S, new, lens, heads, group, dim, P, fmt, elem, seed=case)
    _check_attention(torch, S, c, q, starts, sd, ld, table, max(new), window, causal)


@pytest.mark.gpu
@pytest.mark.parametrize("new", [[1, 1], [90, 150]])
def test_attention_hint_strides_padding(cuda, new):
    torch = cuda
    from hxq_b200 import serving as S
    c, q, starts, sd, ld, table = _attention_case(torch, S, new, [130, 260], 2, 4, 128, 16, "int8", "bf16")
    o, lse = _check_attention(torch, S, c, q, starts, sd, ld, table, max(new))
    for hint in (0, 1, 10 ** 6):   # any value holds
        _check_attention(torch, S, c, q, starts, sd, ld, table, hint)
    # q as a slice of a wider projection, out with strides of its own, rows behind the last request untouched
    T, pad = q.shape[0], 5
    wide = torch.zeros((T + pad, 12, 128), dtype=q.dtype, device="cuda")
    wide[:T, 2:10] = q
    out = torch.full((T + pad, 8, 131), 9.0, dtype=q.dtype, device="cuda")
    lse2 = torch.full((T + pad, 8), 9.0, device="cuda")
    c.attention(wide[:, 2:10], sd, ld, table, max(new), out=out[..., :128], lse=lse2)
    assert torch.equal(out[:T, :, :128], o) and bool((out[T:] == 9).all()) and bool((out[..., 128:] == 9).all())
    assert torch.equal(lse2[:T], lse) and bool((lse2[T:] == 9).all())
    # rows that are not 16-byte aligned are copied
    off = torch.empty(q.numel() + 1, dtype=q.dtype, device="cuda")[1:].view(q.shape)
    off.copy_(q)
    assert torch.equal(c.attention(off, sd, ld, table, max(new)), o)


@pytest.mark.gpu
@pytest.mark.parametrize("new", [[1, 1, 1], [100, 80, 90]])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_attention_extremes(cuda, fmt, new):
    torch = cuda
    from hxq_b200 import serving as S
    lens = [200, 333, 150]
    c, q, starts, sd, ld, table = _attention_case(torch, S, new, lens, 2, 3, 64, 16, fmt, "bf16", spread=3.0)
    q *= torch.exp2(torch.randint(-40, 4, (q.shape[0], q.shape[1], 1), device="cuda").float()).to(q.dtype)
    c.v_scales[table[0, 3].long()] = 0          # a block of zeros among the values
    c.k_scales[table[0, 5].long()] = 0          # and among the keys
    c.v_scales[table[1, 2].long()] = 1e-35      # counts as zero
    c.v_scales[table[2].clamp(min=0)[:3].long()] = 1e30
    _check_attention(torch, S, c, q, starts, sd, ld, table, max(new))
    # all values zero
    c.v_scales.zero_()
    o = c.attention(q, sd, ld, table, max(new))
    assert bool((o == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("new,what", [([2, 1], "k"), ([2, 1], "v"), ([150, 90], "k"), ([150, 90], "v"), ([150, 90], "vinf"), ([150, 90], "q")])
def test_attention_nan_stays_where_it_is_seen(cuda, new, what):
    torch = cuda
    from hxq_b200 import serving as S
    lens = [150, 120]
    c, q, starts, sd, ld, table = _attention_case(torch, S, new, lens, 2, 2, 128, 16, "int8", "bf16")
    clean = c.attention(q, sd, ld, table, max(new))
    blk = lens[0] // 16 - 1                       # a block that the last rows of request 0 see
    first = blk * 16
    if what == "q":
        q[0, 1, 5] = math.nan
        o = c.attention(q, sd, ld, table, max(new))
        assert bool(o[0, 1].isnan().all())
        o[0, 1] = clean[0, 1]
        assert torch.equal(o, clean)
        return
    s = c.k_scales if what == "k" else c.v_scales
    s[table[0, blk].long(), 0] = math.inf if what == "vinf" else math.nan
    o = c.attention(q, sd, ld, table, max(new))
    pos = torch.arange(lens[0] - new[0], lens[0], device="cuda")
    sees = torch.zeros((q.shape[0],), dtype=torch.bool, device="cuda")
    sees[:new[0]] = pos >= first
    assert bool(o[sees][:, :2].isnan().all())
    keep = torch.ones(o.shape[:2], dtype=torch.bool, device="cuda")
    keep[:, :2] = ~sees[:, None]
    assert torch.equal(o[keep], clean[keep])


@pytest.mark.gpu
def test_attention_records_what_is_out_of_range(cuda):
    torch = cuda
    from hxq_b200 import serving as S
    for new in ([1, 1], [80, 70]):
        c, q, starts, sd, ld, table = _attention_case(torch, S, new, [100, 90], 1, 2, 64, 16, "int8", "bf16")
        good = c.attention(q, sd, ld, table, max(new))
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        for entry in (-1, c.n_blocks, 2 ** 31 - 1):
            bad = table.clone()
            bad[0, 1] = entry
            status.zero_()
            o = c.attention(q, sd, ld, bad, max(new), status=status)
            assert int(status) == 2 and torch.equal(o[new[0]:], good[new[0]:]) and bool(o.isfinite().all())
        for s, l, bits in ((sd + 1, ld, 4), (sd, ld + 5000, 2), (sd, ld * 0 - 1, 4), (sd.flip(0).contiguous(), ld, 4)):
            status.zero_()
            o = c.attention(q, s.contiguous(), l.contiguous(), table, max(new), status=status)
            torch.cuda.synchronize()
            assert int(status) & bits, (bits, S.problems(status))


@pytest.mark.gpu
def test_attention_replayed_with_other_lengths(cuda):
    torch = cuda
    from hxq_b200 import serving as S
    c, q, starts, sd, ld, table = _attention_case(torch, S, [1, 1, 1], [900, 30, 500], 2, 4, 128, 16, "int8", "bf16")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c.attention(q, sd, ld, table, 1)
    graphs = []
    for _ in range(2):   # two graphs of the same stream, replayed at once on two streams
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            o = c.attention(q, sd, ld, table, 1)
        graphs.append((g, o))
    for lens in ([900, 30, 500], [17, 800, 1], [1, 1, 1]):
        ld.copy_(torch.tensor(lens, dtype=torch.int32))
        tb = table
        want, _, tol, _ = _attention_ref(torch, c, q, starts, [min(n, m) for n, m in zip(lens, [900, 30, 500])], tb, 128 ** -0.5, 0, True)
        ld.copy_(torch.tensor([min(n, m) for n, m in zip(lens, [900, 30, 500])], dtype=torch.int32))
        torch.cuda.synchronize()
        other = torch.cuda.Stream()
        with torch.cuda.stream(other):
            graphs[0][0].replay()
        graphs[1][0].replay()
        torch.cuda.synchronize()
        for _, o in graphs:
            assert bool(((o.double() - want).abs() <= tol).all()), lens


@pytest.mark.gpu
def test_attention_long_cache_offsets(cuda):
    """Blocks whose byte offset passes 2^32."""
    torch = cuda
    from hxq_b200 import serving as S
    n_blocks = (1 << 32) // (8 * 16 * 128) + 40
    c = S.KvCache.allocate(n_blocks, 8, 128, 16)
    table = torch.arange(n_blocks - 20, n_blocks, dtype=torch.int32, device="cuda").view(2, 10)
    lens, starts = [150, 160], [0, 1, 2]
    plan = torch.cat([table[b].repeat_interleave(16)[:n] * 16 + torch.arange(n, device="cuda") % 16 for b, n in enumerate(lens)]).int()
    x = torch.randn((2, 310, 8, 128), device="cuda").to(torch.bfloat16)
    c.append(x[0], x[1], plan)
    k, _ = c.read(plan, torch.float32)
    assert float((k - x[0].float()).abs().max()) < 0.03
    q = torch.randn((2, 16, 128), device="cuda").to(torch.bfloat16)
    i = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    _check_attention(torch, S, c, q, starts, i(starts), i(lens), table, 1)


# -- adapters ------------------------------------------------------------------------

def _lora_ref(torch, y, x, a, b, scales, starts, ids, I, R):
    out, tol = y.double().clone(), y.double().abs() * 2.0 ** -23
    for r, ad in enumerate(ids):
        if 0 <= ad < a.shape[0]:
            s = slice(starts[r], starts[r + 1])
            aa, bb, sc, xx = a[ad].double(), b[ad].double(), scales[ad].double(), x[s].double()
            out[s] += sc * (xx @ aa.T @ bb.T)
            size = sc.abs() * (xx.abs() @ aa.abs().T @ bb.abs().T)
            # two bf16 parts of h: 2^-17; fp32 sums, 16 products a step, 2^-23 each step
            tol[s] += size * (2.0 ** -17 + (I / 16 + R / 8 + 80) * 2.0 ** -23)
    return out, tol


@pytest.mark.gpu
@pytest.mark.parametrize("new,ids,n,R,I,O", [
    ([1], [0], 1, 8, 64, 8), ([1] * 64, [i % 16 for i in range(64)], 16, 16, 4096, 4096), ([1, 1, 1], [-1, -1, -1], 2, 16, 256, 64),
    ([1, 0, 3, 2], [1, 0, -1, 1], 3, 24, 520, 77), ([100, 3, 70], [2, 0, 2], 4, 64, 1000, 513), ([5, 9], [0, 1], 2, 128, 264, 130),
    ([300, 17, 1, 1], [0, 1, -1, 0], 2, 32, 11008, 256), ([64, 64, 65], [0, 1, 0], 2, 40, 128, 64), ([700], [0], 1, 16, 192, 1024),
    ([2] * 200, [(i * 7) % 33 - 1 for i in range(200)], 40, 8, 64, 40)])
def test_lora(cuda, new, ids, n, R, I, O):
    torch = cuda
    from hxq_b200 import serving as S
    g = torch.Generator().manual_seed(R + I)
    starts = [sum(new[:b]) for b in range(len(new) + 1)]
    T = starts[-1]
    x = torch.randn((T, I), generator=g).to(torch.bfloat16).cuda()
    a = (torch.randn((n, R, I), generator=g) / math.sqrt(I)).to(torch.bfloat16).cuda()
    b = torch.randn((n, O, R), generator=g).to(torch.bfloat16).cuda()
    sc = (torch.randn((n,), generator=g)).cuda()
    y = torch.randn((T, O), generator=g).cuda()
    i = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    status = i([0])
    plan = S.lora_plan(i(starts), i(ids), n, T, status=status)
    # the plan: every token once, tiles of one adapter, in order
    order, seen = plan.order.tolist(), []
    of = [ad for ad, k in zip(ids, new) for _ in range(k)]
    for ad, first, count, _ in plan.tiles.tolist():
        assert 0 <= count <= 64
        if count:
            assert all(of[t] == ad for t in order[first:first + count])
            seen += order[first:first + count]
    assert seen == sorted(range(T), key=lambda t: (of[t] if of[t] >= 0 else n, t))
    h = S.LoraAdapters(a, b, sc)
    out = h.add(y, x, plan)
    want, tol = _lora_ref(torch, y, x, a, b, sc, starts, ids, I, R)
    over = (out.double() - want).abs() - tol
    assert int(status) == 0 and bool((over <= 0).all()), float(over.max())
    assert torch.equal(h.add(y, x, plan), out)
    # in place, on slices of wider rows, with rows behind the last request
    wx = torch.zeros((T + 3, I + 8), dtype=torch.bfloat16, device="cuda")
    wx[:T, :I] = x
    wy = torch.full((T + 3, O + 1), 5.0, device="cuda")
    wy[:T, :O] = y
    wide = S.lora_plan(i(starts), i(ids), n, T + 3)
    got = h.add(wy[:, :O], wx[:, :I], wide, out=wy[:, :O])
    assert got.data_ptr() == wy.data_ptr()
    over = (wy[:T, :O].double() - want).abs() - tol
    assert bool((over <= 0).all()) and bool((wy[T:] == 5).all()) and bool((wy[:, O] == 5).all())


@pytest.mark.gpu
def test_lora_bad_numbers(cuda):
    torch = cuda
    from hxq_b200 import serving as S
    i = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    x, y = torch.randn(4, 64, device="cuda").to(torch.bfloat16), torch.randn(4, 32, device="cuda")
    a, b = torch.randn(2, 8, 64, device="cuda").to(torch.bfloat16), torch.randn(2, 32, 8, device="cuda").to(torch.bfloat16)
    h, status = S.LoraAdapters(a, b, torch.ones(2, device="cuda")), i(0)
    plan = S.lora_plan(i(0, 1, 3, 4), i(7, -5, 2), 2, 4, status=status)   # no adapter 7 or 2
    assert int(status) == 32 and torch.equal(h.add(y, x, plan), y)
    for starts in (i(0, 9, 4, 4), i(3, 1, 4, 4), i(-2, 4, 0, 4)):
        status.zero_()
        plan = S.lora_plan(starts, i(0, 1, 0), 2, 4, status=status)
        h.add(y, x, plan)
        torch.cuda.synchronize()
        assert int(status) == 4


# -- a step of all of them --------------------------------------------------------------

@pytest.mark.gpu
def test_serving_step(H, L, cuda):
    """Two steps of a small layer on compressed projections: plan, projections
    with adapters, rotation, append, attention; captured and replayed."""
    torch = cuda
    from hxq_b200 import serving as S, synth
    from hxq_b200.torch_ops import HxqLinear
    hidden, heads, kvh, D, P = 512, 4, 2, 64, 16
    wq, wk, wv = (HxqLinear(synth.vq12(o, hidden, 50 + s)) for s, o in enumerate((heads * D, kvh * D, kvh * D)))
    g = torch.Generator().manual_seed(9)
    la = S.LoraAdapters((torch.randn((2, 8, hidden), generator=g) / 20).to(torch.bfloat16).cuda(),
                        torch.randn((2, heads * D, 8), generator=g).to(torch.bfloat16).cuda(), torch.ones(2, device="cuda"))
    rot = torch.empty(D * D, dtype=torch.float32)
    assert L.pq_generate_rotation(D, 4, rot.data_ptr()) == 0
    rot = rot.cuda()
    cache = S.KvCache.allocate(40, kvh, D, P)
    free, table = torch.randperm(40, generator=g).to(torch.int32).cuda(), torch.full((3, 8), -1, dtype=torch.int32, device="cuda")
    ids = torch.tensor([1, -1, 0], dtype=torch.int32, device="cuda")
    state = {}

    def step(x, new, cached, free, max_new):
        plan = S.kv_plan(new, cached, table, free, P, x.shape[0])
        lp = S.lora_plan(plan.starts, ids, 2, x.shape[0])
        q = wq(x, adapters=la, plan=lp).view(-1, heads, D)
        k, v = wk(x).view(-1, kvh, D), wv(x).view(-1, kvh, D)
        state.update(q=q.clone(), k=k.clone(), v=v.clone(), plan=plan)
        for t in (q, k):   # scores don't change: both are rotated
            H.check(L.hxq_cuda_pq_rotate(t.data_ptr(), rot.data_ptr(), t.numel() // D, D, torch.cuda.current_stream().cuda_stream))
        cache.append(k, v, plan.slots)
        return cache.attention(q.to(torch.bfloat16), plan.starts, plan.lens, table, max_new)

    i = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    hist = [[], [], []]

    def check(o, new, x):
        assert torch.allclose(state["q"], wq(x).view(-1, heads, D), atol=0) is False   # the adapters did something
        at = 0
        for b, n in enumerate(new):
            hist[b] += [(state["k"][at + t].clone(), state["v"][at + t].clone()) for t in range(n)]   # the graph reuses them
            K, V = (torch.stack([h[w] for h in hist[b]]).double() for w in (0, 1))
            for t in range(n):
                m = len(hist[b]) - n + t + 1
                for h in range(heads):
                    kk, vv = K[:m, h // 2], V[:m, h // 2]
                    qq = state["q"][at + t, h].double()
                    p = torch.softmax(kk @ qq / 8, 0)
                    want = p @ vv
                    # a block's largest value sets its step; keys move scores, values the sum; q and out are bf16
                    step_k, step_v = kk.abs().max() * 8 / 127, vv.abs().max() / 127
                    ds = (qq.norm() * step_k * 0.5 + kk.norm(dim=1).max() * qq.norm() * 2.0 ** -8) / 8
                    tol = step_v + 2 * torch.expm1(2 * ds) * (p @ vv.abs()).max() + 2.0 ** -7 * want.abs().max()
                    assert float((o[at + t, h].double() - want).abs().max()) <= float(tol)
            at += n

    x0 = torch.randn((30, hidden), generator=g).to(torch.bfloat16).cuda()
    o = step(x0, i(5, 20, 5), i(0, 0, 0), free, 20)
    check(o, [5, 20, 5], x0)
    # decode steps: one graph, replayed with the lengths that follow
    x1, cached, used = torch.randn((3, hidden), generator=g).to(torch.bfloat16).cuda(), i(5, 20, 5), int(state["plan"].taken)
    fl = free[used:].clone()
    one = i(1, 1, 1)
    snap = [t.clone() for t in (cache.k, cache.v, cache.k_scales, cache.v_scales, table)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x1, one, cached, fl, 1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        o = step(x1, one, cached, fl, 1)
    for t, s in zip((cache.k, cache.v, cache.k_scales, cache.v_scales, table), snap):
        t.copy_(s)
    for n in range(14):
        x1.copy_(torch.randn((3, hidden), generator=g).to(torch.bfloat16))
        graph.replay()
        check(o, [1, 1, 1], x1)
        taken = int(state["plan"].taken)
        fl.copy_(torch.cat([fl[taken:], fl[:taken]]))
        cached += 1


# -- calls that programs make in other ways ----------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("new_most", [1, 70])
def test_attention_many_requests(cuda, new_most):
    """Thousands of short requests, some empty: more than threads, several to a CTA."""
    torch = cuda
    from hxq_b200 import serving as S
    g = torch.Generator().manual_seed(new_most)
    B = 2500 if new_most == 1 else 300
    new = [new_most if i % 50 == 7 else 1 for i in range(B)]
    lens = [int(v) if i % 11 else 0 for i, v in enumerate(torch.randint(1, 60, (B,), generator=g))]
    lens = [max(n, m) if n else 0 for n, m in zip(lens, new)]
    c, q, starts, sd, ld, table = _attention_case(torch, S, new, lens, 1, 2, 64, 16, "int8", "bf16", seed=new_most)
    _check_attention(torch, S, c, q, starts, sd, ld, table, new_most)


@pytest.mark.gpu
def test_calls_on_two_streams_at_once(cuda):
    torch = cuda
    from hxq_b200 import serving as S
    cases = [_attention_case(torch, S, new, lens, 2, 4, 128, 16, fmt, "bf16", seed=s)
             for s, (new, lens, fmt) in enumerate((([1, 1], [3000, 900], "int8"), ([300, 20], [700, 2000], "e4m3")))]
    want = [c.attention(q, sd, ld, t, 300) for c, q, _, sd, ld, t in cases]
    g = torch.Generator().manual_seed(1)
    a = torch.randn((3, 16, 512), generator=g).to(torch.bfloat16).cuda()
    b = torch.randn((3, 640, 16), generator=g).to(torch.bfloat16).cuda()
    h = S.LoraAdapters(a, b, torch.ones(3, device="cuda"))
    x, y = torch.randn((90, 512), generator=g).to(torch.bfloat16).cuda(), torch.randn((90, 640), generator=g).cuda()
    i = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    starts, ids = i([0, 40, 41, 90]), i([2, -1, 0])
    added = h.add(y, x, S.lora_plan(starts, ids, 3, 90))
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(3)], [[], [], []]
    for _ in range(5):
        for k, (c, q, _, sd, ld, t) in enumerate(cases):
            with torch.cuda.stream(streams[k]):
                got[k].append(c.attention(q, sd, ld, t, 300))
        with torch.cuda.stream(streams[2]):
            got[2].append(h.add(y, x, S.lora_plan(starts, ids, 3, 90)))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[k]) for k in range(2) for o in got[k]) and all(torch.equal(o, added) for o in got[2])


@pytest.mark.gpu
def test_lora_replayed_with_other_requests(cuda):
    torch = cuda
    from hxq_b200 import serving as S
    g = torch.Generator().manual_seed(4)
    n, R, I, O, T = 4, 24, 256, 96, 50
    a = (torch.randn((n, R, I), generator=g) / 16).to(torch.bfloat16).cuda()
    b, sc = torch.randn((n, O, R), generator=g).to(torch.bfloat16).cuda(), torch.ones(n, device="cuda")
    x, y = torch.randn((T, I), generator=g).to(torch.bfloat16).cuda(), torch.randn((T, O), generator=g).cuda()
    h = S.LoraAdapters(a, b, sc)
    starts, ids = torch.tensor([0, 50, 50, 50], dtype=torch.int32, device="cuda"), torch.tensor([0, 0, 0], dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        h.add(y, x, S.lora_plan(starts, ids, n, T))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = h.add(y, x, S.lora_plan(starts, ids, n, T))
    for st, ad in (([0, 50, 50, 50], [0, 1, 2]), ([0, 7, 30, 50], [3, -1, 3]), ([0, 1, 2, 3], [1, 2, 0])):
        starts.copy_(torch.tensor(st, dtype=torch.int32))
        ids.copy_(torch.tensor(ad, dtype=torch.int32))
        out.fill_(8.0)
        graph.replay()
        torch.cuda.synchronize()
        want, tol = _lora_ref(torch, y, x, a, b, sc, st, ad, I, R)
        assert bool(((out.double() - want).abs() <= tol)[:st[-1]].all()) and bool((out[st[-1]:] == 8).all())


@pytest.mark.gpu
def test_empty_calls(cuda):
    torch = cuda
    from hxq_b200 import serving as S
    i = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    c = S.KvCache.allocate(4, 2, 64)
    none = torch.zeros((0, 2, 64), device="cuda")
    c.append(none, none, i())
    assert c.read(i())[0].shape == (0, 2, 64)
    q = torch.zeros((0, 2, 64), dtype=torch.bfloat16, device="cuda")
    assert c.attention(q, i(0), i(), torch.zeros((0, 1), dtype=torch.int32, device="cuda"), 1).shape == q.shape
    q = torch.full((3, 2, 64), 2.0, dtype=torch.bfloat16, device="cuda")
    out = q.clone()
    c.attention(q, i(0, 0, 0), i(5, 0), torch.zeros((2, 1), dtype=torch.int32, device="cuda"), 1, out=out)   # no rows of any request
    assert bool((out == 2).all())
    h = S.LoraAdapters(torch.zeros((1, 8, 64), dtype=torch.bfloat16, device="cuda"), torch.zeros((1, 32, 8), dtype=torch.bfloat16, device="cuda"),
                       torch.ones(1, device="cuda"))
    assert h.add(torch.zeros((0, 32), device="cuda"), torch.zeros((0, 64), dtype=torch.bfloat16, device="cuda"), S.lora_plan(i(0), i(), 1, 0)).shape == (0, 32)


@pytest.mark.gpu
@pytest.mark.parametrize("R", [8, 32])
def test_lora_infinity(cuda, R):
    # an infinity in a row of x gives that row infinities (NaN where B is
    # zero), as the formula does, and nothing in another row
    torch = cuda
    from hxq_b200 import serving as S
    T, I, O = 5, 64, 24
    g = torch.Generator("cuda").manual_seed(3)
    x = torch.randn(T, I, device="cuda", generator=g).bfloat16()
    x[2, 5] = float("inf")
    a = torch.rand(1, R, I, device="cuda", generator=g).bfloat16() + 1
    b = torch.rand(1, O, R, device="cuda", generator=g).bfloat16() + 1
    b[0, 3] = 0
    b[0, 7] = -b[0, 7]
    y = torch.zeros(T, O, device="cuda")
    starts = torch.tensor([0, T], dtype=torch.int32, device="cuda")
    ids = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = S.LoraAdapters(a, b, torch.ones(1, device="cuda")).add(y, x, S.lora_plan(starts, ids, 1, T))
    want = (x.double() @ a[0].double().T) @ b[0].double().T
    assert torch.equal(torch.isnan(out), torch.isnan(want)) and bool(torch.isnan(out[2, 3]))
    assert bool((out[2][torch.isinf(want[2])] == want[2][torch.isinf(want[2])].float()).all())
    assert bool(torch.isfinite(out[[0, 1, 3, 4]]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new,lens,heads,group,window,causal", [
    ([100], [1500], 2, 1, 0, True),                                  # one tile of rows, many steps
    ([129, 257, 300, 65], [129, 2000, 5000, 4000], 4, 1, 0, True),   # two tiles, the second with fewer rows
    ([300, 90], [2500, 90], 8, 5, 700, True),
    ([300, 100], [900, 1000], 2, 3, 0, False),
    ([150, 70] * 12, [400, 130] * 12, 8, 1, 0, True),                # many units a CTA, of one tile and of two
])
def test_attention_tiles_of_rows(cuda, dim, new, lens, heads, group, window, causal):
    torch = cuda
    from hxq_b200 import serving as S
    c, q, starts, sd, ld, table = _attention_case(torch, S, new, lens, heads, group, dim, 32, "e4m3", "bf16", seed=len(new))
    _check_attention(torch, S, c, q, starts, sd, ld, table, max(new), window, causal)


@pytest.mark.gpu
@pytest.mark.parametrize("new,lens,heads,group,window", [
    ([256, 100], [6000, 3000], 8, 1, 0), ([130] * 6, [2600] * 6, 4, 5, 700), ([512, 512], [8704, 8192], 4, 5, 4096)])
def test_attention_maxima_of_a_rows_halves(cuda, new, lens, heads, group, window):
    """Heads of 64, where the next scores of a tile are there while its warps
    are at these: keys that grow all the way, so that the maximum of both
    halves of a row is raised in most steps, and the same bits every time."""
    torch = cuda
    from hxq_b200 import serving as S
    c, q, starts, sd, ld, table = _attention_case(torch, S, new, lens, heads, group, 64, 16, "int8", "bf16", seed=len(new), spread=0.3)
    for b, n in enumerate(lens):
        pages = table[b, :-(-n // 16)].long()
        c.k_scales[pages] *= torch.exp2(torch.arange(len(pages), device="cuda") * (6.0 / len(pages)))[:, None]
    o, _ = _check_attention(torch, S, c, q, starts, sd, ld, table, max(new), window)
    for _ in range(30):
        assert torch.equal(c.attention(q, sd, ld, table, max(new), window=window), o)


@pytest.mark.gpu
@pytest.mark.parametrize("cycles", [0, 300, 1500, 4000, 10000, 25000])
@pytest.mark.parametrize("dim,new,lens", [
    (64, [1, 1], [2500, 1200]), (128, [1, 3], [2500, 1200]), (64, [300, 90], [2500, 1200]), (128, [300, 90], [2500, 1200]),
    (64, [1, 1], [200000, 150000]), (128, [2, 1], [200000, 150000])])
def test_attention_waits_that_run_out(H, L, cuda, dim, new, lens, cycles):
    """A wait inside the kernels that runs out ends the call with a status,
    wherever it is, and the next call is as if nothing had been."""
    torch = cuda
    from hxq_b200 import serving as S
    c, q, starts, sd, ld, table = _attention_case(torch, S, new, lens, 4, 2, dim, 16, "int8", "bf16")
    clean = c.attention(q, sd, ld, table, max(new))
    torch.cuda.synchronize()
    L.hxq_serving_wait_cycles.argtypes, L.hxq_serving_wait_cycles.restype = [C.c_uint32], C.c_uint32
    before = L.hxq_serving_wait_cycles(cycles)
    try:
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        o = c.attention(q, sd, ld, table, max(new), status=status)
        torch.cuda.synchronize()
    finally:
        assert L.hxq_serving_wait_cycles(before) == cycles
    assert before > 10 ** 9 and int(status) in (0, 64)
    assert int(status) == 64 or torch.equal(o, clean)
    assert int(status) == 64 or cycles   # without any patience no call ends as it should
    status.zero_()
    assert torch.equal(c.attention(q, sd, ld, table, max(new), status=status), clean) and int(status) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("B,T,heads,max_new", [(64, 40, 4, 1), (64, 40, 4, 40), (8192, 1 << 17, 64, 1), (8192, 1 << 17, 64, 1 << 17)])
def test_attention_overlapping_requests(cuda, B, T, heads, max_new):
    """Starts 0, T, 0, T, ..: far more rows than there are (in the last two
    shapes 2^32 tiles and more), recorded and not worked off."""
    torch = cuda
    from hxq_b200 import serving as S
    c = S.KvCache.allocate(4, 1, 64)
    q = torch.ones((T, heads, 64), dtype=torch.bfloat16, device="cuda")
    starts = torch.tensor([T * (b & 1) for b in range(B + 1)], dtype=torch.int32, device="cuda")
    lens = torch.full((B,), 17, dtype=torch.int32, device="cuda")
    table = torch.zeros((B, 2), dtype=torch.int32, device="cuda")
    out, status = torch.full_like(q, 9.0), torch.zeros(1, dtype=torch.int32, device="cuda")
    c.attention(q, starts, lens, table, max_new, causal=False, out=out, status=status)
    torch.cuda.synchronize()
    # a cache of zeros: a request's result is 0
    assert int(status) == 4 and bool(((out == 9) | (out == 0)).all()) and (B < 8192 or bool((out == 9).all()))


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("new,lens,heads,group,dim,P,window", [
    ([1, 2], [300, 77], 2, 4, 128, 16, 40), ([1], [1000], 1, 1, 64, 16, 3), ([1, 3], [500, 129], 1, 8, 256, 32, 100),
    ([5, 4], [90, 400], 2, 3, 64, 16, 1), ([100, 90], [700, 400], 2, 3, 64, 16, 50), ([300, 70], [1000, 1111], 1, 2, 128, 16, 333),
    ([129], [129 + 640], 2, 1, 128, 128, 511), ([150, 80] * 4, [900, 700] * 4, 4, 2, 64, 64, 130)])
def test_attention_blocks_behind_the_window(cuda, fmt, new, lens, heads, group, dim, P, window):
    """A program frees blocks that a window has passed: their entries are no
    blocks, and slots that no row sees hold anything, NaN codes among it."""
    torch = cuda
    from hxq_b200 import serving as S
    c, q, starts, sd, ld, table = _attention_case(torch, S, new, lens, heads, group, dim, P, fmt, "bf16", seed=window)
    clean, _ = _check_attention(torch, S, c, q, starts, sd, ld, table, max(new), window)
    for b, (m, n) in enumerate(zip(new, lens)):
        first = max(n - m - window + 1, 0)   # the first key that a row sees
        for j in range(first // P):
            c.k_scales[table[b, j].long()] = math.nan
            c.v_scales[table[b, j].long()] = math.nan
            table[b, j] = (-1, c.n_blocks, 2 ** 31 - 1)[j % 3]
        if first % P:
            c.k.view(torch.uint8)[table[b, first // P].long(), :, :first % P] = 0x7f
            c.v.view(torch.uint8)[table[b, first // P].long(), :, :first % P] = 0xff
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    o = c.attention(q, sd, ld, table, max(new), window=window, status=status)
    assert int(status) == 0 and torch.equal(o, clean)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("new,n,B,heads,dim", [(1, 8192, 74, 8, 64), (1, 8192, 74, 8, 128), (130, 16384, 5, 32, 64), (130, 16384, 5, 32, 128)])
def test_attention_key_that_takes_the_weight(cuda, new, n, B, heads, dim, fmt):
    """A first key with nearly all of the weight and a value of 0, as trained
    models have it: what is left is a sum over the others, each 2^-23 of it."""
    torch = cuda
    from hxq_b200 import serving as S
    g = torch.Generator("cuda").manual_seed(dim)
    P, top = 64, QMAX[fmt]
    n_blocks = B * n // P
    c = S.KvCache.allocate(n_blocks, heads, dim, P, _types(torch)[fmt])
    sign = torch.randint(0, 2, (dim,), generator=g, device="cuda") * 2.0 - 1
    for t in (c.k, c.v):
        x = torch.randn(t.shape, generator=g, device="cuda").mul_(0.3).clamp_(-1, 1) * top
        t.view(torch.int8).copy_((x.round() if fmt == "int8" else x).to(t.dtype).view(torch.int8))
    table = torch.arange(n_blocks, dtype=torch.int32, device="cuda").view(B, -1)
    c.k.view(torch.int8)[table[:, 0].long(), :, 0] = (sign * top).to(c.k.dtype).view(torch.int8)
    c.v.view(torch.int8)[table[:, 0].long(), :, 0] = 0
    c.k_scales.fill_(1 / top)
    c.v_scales.fill_(1024 / top)   # what is left of the sum stays among f16's normal numbers
    # score of the first key: log of (number of keys x 999) above the others' mean
    beta = math.log(n * 999) / math.sqrt(dim)
    q = (sign * beta * (1 + 0.002 * torch.randn((B * new, heads, 1), generator=g, device="cuda"))).to(torch.float16)
    i = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    lse = torch.zeros(q.shape[:2], device="cuda")
    o = c.attention(q, i([b * new for b in range(B + 1)]), i([n] * B), table, new, causal=False, lse=lse)
    for b, h, t in ((0, 0, 0), (B - 1, heads - 1, new - 1), (B // 2, 3, new // 2)):
        k, v = (x[table[b].long(), h].double().reshape(-1, dim) * float(s[0, 0]) for x, s in ((c.k, c.k_scales), (c.v, c.v_scales)))
        sc = k @ q[b * new + t, h].double() / math.sqrt(dim)
        p = torch.softmax(sc, 0)
        assert 0.99 < float(p[0]) < 0.9999
        want = p @ v
        # A weight is rounded by up to 2^-11 of it or 2^-32 of the first key's, evenly spread, so the deviation of the sum
        # over values of mean 0 is at most 2^-11 / sqrt(3) + (2^-32 / sqrt(3)) / (0.0001 / n) of its own: 0.03% + 0.22% and,
        # for 16,384 keys of which p[0] leaves least, + 0.44%; out is rounded by 2^-12. Three deviations: 1.5%.
        rms = float((o[b * new + t, h].double() - want).norm() / want.norm())
        assert rms < 0.015, (b, h, t, rms)
        assert abs(float(lse[b * new + t, h]) - float(torch.logsumexp(sc, 0))) < 1e-4


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("new", [[1, 1, 1], [100, 80, 90]])
@pytest.mark.parametrize("exponent", [127, 120, 116, 115, -86, -100, -118])
def test_attention_queries_near_the_ends_of_bf16(cuda, exponent, new, dim):
    """Rows of q that f16 cannot hold by far, with scales that bring the scores
    back to the ordinary."""
    torch = cuda
    from hxq_b200 import serving as S
    c, q, starts, sd, ld, table = _attention_case(torch, S, new, [200, 333, 150], 2, 3, dim, 16, "int8", "bf16", spread=0.3)
    q = (q.float() / q.float().abs().amax(-1, keepdim=True) * 1.98).to(torch.bfloat16)
    q = (q.float() * 2.0 ** (exponent // 2) * 2.0 ** (exponent - exponent // 2)).to(torch.bfloat16)
    assert bool(q.isfinite().all())
    to_keys = min(exponent, 100)   # the rest, which key scales cannot take, to the factor of the scores
    c.k_scales.mul_(2.0 ** -to_keys)
    assert bool((c.k_scales > 2.0 ** -126).all()) and bool(c.k_scales.isfinite().all())
    _check_attention(torch, S, c, q, starts, sd, ld, table, max(new), scale=dim ** -0.5 * 2.0 ** (to_keys - exponent))


_FIRST_CALL = """
import sys
sys.path.insert(0, {pkg!r})
import torch
from hxq_b200 import serving as S
B, n = {B}, {n}
i = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
status = i([0])
if {op!r} == "plan":
    p = S.kv_plan(i([1] * B), i([0] * B), i([-1] * B).view(B, 1), i(list(range(B))), 16, B, status=status)
    assert p.slots.tolist() == [16 * b for b in range(B)] and int(p.taken) == B
else:
    p = S.lora_plan(i(list(range(B + 1))), i([b % n for b in range(B)]), n, B, status=status)
    assert p.order.tolist() == sorted(range(B), key=lambda b: b % n)
assert int(status) == 0
"""


@pytest.mark.gpu
@pytest.mark.parametrize("B", [6109, 6110, 6143, 6144])
def test_plan_as_a_process_first_call(cuda, B):
    """Sizes about the limit of shared memory that needs no permission, which
    an earlier and larger call would have raised."""
    import subprocess
    import sys

    from conftest import PKG
    subprocess.run([sys.executable, "-c", _FIRST_CALL.format(pkg=PKG, B=B, n=0, op="plan")], check=True, timeout=120)


@pytest.mark.gpu
@pytest.mark.parametrize("B,n", [(6109, 1), (6110, 1), (6141, 1), (6142, 1), (300, 3894)])
def test_lora_plan_as_a_process_first_call(cuda, B, n):
    import subprocess
    import sys

    from conftest import PKG
    subprocess.run([sys.executable, "-c", _FIRST_CALL.format(pkg=PKG, B=B, n=n, op="lora_plan")], check=True, timeout=120)


@pytest.mark.gpu
def test_tensors_that_move(cuda):
    """Calls use the memory that the tensors have then, not what they had."""
    torch = cuda
    from hxq_b200 import serving as S
    i = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    c = S.KvCache.allocate(4, 2, 64)
    before = [t.detach() for t in (c.k, c.v, c.k_scales, c.v_scales)]
    c.k.data = torch.zeros_like(c.k)
    c.v.set_(torch.zeros_like(c.v))
    c.k_scales.data = torch.zeros_like(c.k_scales)
    c.v_scales.data = torch.zeros_like(c.v_scales)
    x = torch.randn((2, 16, 2, 64), device="cuda")
    c.append(x[0], x[1], torch.arange(16, 32, dtype=torch.int32, device="cuda"))
    assert all(bool((t.float() == 0).all()) for t in before)
    k, v = c.read(torch.arange(16, 32, dtype=torch.int32, device="cuda"), torch.float32)
    assert float((k - x[0]).abs().max()) < 0.03 and float((v - x[1]).abs().max()) < 0.03
    q = torch.randn((1, 2, 64), device="cuda").to(torch.bfloat16)
    o = c.attention(q, i(0, 1), i(16), i(1).view(1, 1), 1)
    want = torch.softmax(torch.einsum("hd,thd->ht", q[0].float(), k) / 8, -1)
    assert float((o[0].float() - torch.einsum("ht,thd->hd", want, v)).abs().max()) < 0.02
    for bad in (lambda: c.k.data.new_zeros((3, 2, 16, 64)), lambda: c.k.data.new_zeros((4, 2, 16, 64)).transpose(0, 1).contiguous().transpose(0, 1),
                lambda: c.k.data.cpu(), lambda: c.k.data.view(torch.float8_e4m3fn)):
        keep, c.k.data = c.k.data, bad()
        for call in (lambda: c.append(x[0], x[1], i(*range(16))), lambda: c.read(i(0)), lambda: c.attention(q, i(0, 1), i(16), i(1).view(1, 1), 1)):
            with pytest.raises(ValueError):
                call()
        c.k.data = keep
    assert torch.equal(c.read(torch.arange(16, 32, dtype=torch.int32, device="cuda"), torch.float32)[0], k)
    with pytest.raises(AttributeError):
        c.k = torch.zeros_like(c.k)

    a, b = torch.randn((2, 8, 64), device="cuda").bfloat16(), torch.randn((2, 32, 8), device="cuda").bfloat16()
    h = S.LoraAdapters(a, b, torch.ones(2, device="cuda"))
    plan = S.lora_plan(i(0, 5), i(1), 2, 5)
    y, xx = torch.zeros((5, 32), device="cuda"), torch.randn((5, 64), device="cuda").bfloat16()
    one = h.add(y, xx, plan)
    a.data, b.data, h.scales.data = a * 2, b * 2, torch.full((2,), 2.0, device="cuda")
    assert torch.equal(h.add(y, xx, plan), one * 8)
    keep, h.b.data = h.b.data, torch.zeros((2, 40, 8), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError):
        h.add(y, xx, plan)
    h.b.data = keep
    with pytest.raises(AttributeError):
        h.a = a


@pytest.mark.gpu
def test_no_gradient_is_lost(H, L, cuda):
    """Calls that would leave their part out of a gradient are refused, and
    what calls write in place counts as changed."""
    torch = cuda
    from hxq_b200 import serving as S, synth
    from hxq_b200.torch_ops import HxqLinear
    i = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    c = S.KvCache.allocate(4, 2, 64)
    kv, table, status = torch.randn((3, 2, 64), device="cuda"), i(-1).view(1, 1), i(0)
    q = torch.randn((3, 2, 64), device="cuda").to(torch.bfloat16)
    out, lse = torch.zeros_like(q), torch.zeros((3, 2), device="cuda")
    a, b = torch.randn((1, 8, 64), device="cuda").bfloat16(), torch.randn((1, 32, 8), device="cuda").bfloat16()
    scales = torch.ones(1, device="cuda")
    h = S.LoraAdapters(a, b, scales)
    x, y = torch.randn((3, 64), device="cuda").bfloat16(), torch.randn((3, 32), device="cuda")
    plan = S.kv_plan(i(3), i(0), table, i(2), 16, 3, status=status)
    lp = S.lora_plan(plan.starts, i(0), 1, 3)
    attend = lambda q, **kw: c.attention(q, plan.starts, plan.lens, table, 3, **kw)  # noqa: E731

    def grad(t):
        return t.detach().clone().requires_grad_()
    calls = [lambda: c.append(grad(kv), kv, plan.slots), lambda: c.append(kv, grad(kv), plan.slots), lambda: attend(grad(q)),
             lambda: attend(q, lse=grad(lse)), lambda: h.add(grad(y), x, lp), lambda: h.add(y, grad(x), lp),
             lambda: S.LoraAdapters(grad(a), b, scales).add(y, x, lp), lambda: S.LoraAdapters(a, grad(b), scales).add(y, x, lp),
             lambda: S.LoraAdapters(a, b, grad(scales)).add(y, x, lp)]
    wide = HxqLinear(synth.scalar(32, 64, 3)), HxqLinear(synth.vq12(32, 64, 4))
    assert [w.fused for w in wide] == [False, True]
    calls += [lambda w=w: w(grad(x), adapters=h, plan=lp) for w in wide]
    before = [t.clone() for t in (c.k, c.k_scales, y)]
    for call in calls:
        with pytest.raises(RuntimeError, match="gradient"):
            call()
    assert all(torch.equal(t, w) for t, w in zip((c.k, c.k_scales, y), before))
    with torch.no_grad():
        for call in calls:
            call()
    # the projection by itself keeps its gradient
    xg = grad(x)
    wide[0](xg).sum().backward()
    assert torch.allclose(xg.grad.float(), wide[0].weight().sum(0).expand(3, -1), rtol=2.0 ** -8, atol=1e-3)

    written = (table, c.k, c.v, c.k_scales, c.v_scales, out, lse, status, y)
    v0 = [t._version for t in written]
    S.kv_plan(i(3), i(0), table, i(2), 16, 3)
    c.append(kv, kv, plan.slots)
    attend(q, out=out, lse=lse, status=status)
    h.add(y, x, lp, out=y)
    assert all(t._version > v for t, v in zip(written, v0))
    w = torch.randn_like(y).requires_grad_()
    z = (w * y).sum()
    h.add(y, x, lp, out=y)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        z.backward()
    # under inference mode, whose tensors count nothing
    with torch.inference_mode():
        ci = S.KvCache.allocate(4, 2, 64)
        ci.append(kv, kv, plan.slots)
    ci.append(kv, kv, plan.slots)
    assert torch.equal(ci.k, c.k)


@pytest.mark.parametrize("kw,code", [
    (dict(out_stride_t=0), 34), (dict(out_stride_h=0), 34), (dict(out_stride_t=255), 34), (dict(out_stride_h=63), 34),
    (dict(out_stride_t=64, out_stride_h=64), 34), (dict(out_stride_t=64, out_stride_h=9 * 64 - 1), 34),
    (dict(out=FAKE + 2), 34), (dict(out=FAKE + 2 * 256 * 3), 34), (dict(out=FAKE - 2 * (256 + 64)), 34),
    (dict(out=FAKE, out_stride_t=512), 34), (dict(out_stride_t=-200), 34),
    (dict(q_stride_t=1024, out_stride_t=1024, out=FAKE + 2 * 255), 34), (dict(q_stride_t=1024, out_stride_t=1024, out=FAKE + 2 * (1024 * 3 - 255)), 34)])
def test_attention_out_has_places_of_its_own(H, L, kw, code):
    d = dict(q=FAKE, out=FAKE + (1 << 30), starts=FAKE, lens=FAKE, table=FAKE, n_requests=1, n_rows=9, n_heads=4, table_width=1,
             max_new=1, scale=1.0, elem=1, causal=1, q_stride_t=256, q_stride_h=64, out_stride_t=256, out_stride_h=64)
    a = H.KvAttention(**{**d, **kw})
    assert L.hxq_cuda_kv_attention(C.byref(_cache(H)), C.byref(a), FAKE, 1 << 40, None, None) == code


def test_overlaps_against_every_element(H, L, tmp_path):
    """The host's arithmetic about strides against the elements themselves."""
    import os
    import subprocess

    from conftest import PKG, REPO
    src = tmp_path / "t.cu"
    src.write_text(r"""
#include "serving_common.cuh"
#include <cstdio>
#include <map>
#include <random>
#include <set>
using hxq::serving::Runs;
int main()
{
    std::mt19937 g(1);
    auto pick = [&](int lo, int hi) { return (int64_t)(lo + (int)(g() % (unsigned)(hi - lo + 1))); };
    long seen[4] = {0, 0, 0, 0};
    for (int k = 0; k < 300000; ++k) {
        Runs w = {(uintptr_t)(1000 + 2 * pick(0, 120)), {pick(1, 4), pick(1, 4)}, {pick(-30, 30), pick(-30, 30)}, pick(1, 6), 2};
        Runs r = w;
        r.at = (uintptr_t)(1000 + 2 * pick(0, 120));
        if (pick(0, 2) == 0) { r.stride[0] = pick(-30, 30); r.stride[1] = pick(-30, 30); }
        auto elements = [](const Runs &x, bool &twice) {
            std::map<long, int> e;
            int at = 0;
            for (int64_t i = 0; i < x.n[0]; ++i)
                for (int64_t j = 0; j < x.n[1]; ++j)
                    for (int64_t d = 0; d < x.width; ++d)
                        if (!e.emplace((long)x.at + 2 * (i * x.stride[0] + j * x.stride[1] + d), at++).second) twice = true;
            return e;
        };
        bool twice = false, ignore = false;
        const auto a = elements(w, twice), b = elements(r, ignore);
        if (w.apart()) {
            if (twice) { std::printf("apart, but twice\n"); return 1; }
            bool share = false, same = a == b;
            for (auto &x : a) share |= b.count(x.first) != 0;
            const bool ok = w.may_overwrite(r);
            if (ok && share && !same) { std::printf("shared and not the same\n"); return 2; }
            bool strides = true;
            for (int d = 0; d < 2; ++d) strides &= w.n[d] == 1 || w.stride[d] == r.stride[d];
            if (!ok && strides && (!share || same)) { std::printf("refused without need\n"); return 3; }
            ++seen[ok ? (share ? 0 : 1) : 2];
        } else ++seen[3];
    }
    for (long s : seen) if (s < 100) { std::printf("too few of a kind\n"); return 4; }
    return 0;
}
""")
    nvcc = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
    if not os.path.exists(nvcc):
        pytest.skip("no nvcc")
    exe = tmp_path / "t"
    subprocess.run([nvcc, "-std=c++17", "-arch=sm_100a", "-I", os.path.join(REPO, "include"), "-I", os.path.join(PKG, "csrc"), str(src), "-o", str(exe)],
                   check=True, capture_output=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout


def test_lora_out_has_places_of_its_own(H, L):
    def call(y=FAKE, ldy=48, out=FAKE + (1 << 30), ldo=48):
        l = H.LoraDesc(a=FAKE, b=FAKE, scales=FAKE, n_adapters=2, rank=16, in_features=64, out_features=48)
        return L.hxq_cuda_lora(C.byref(l), FAKE, 64, y, ldy, out, ldo, 2, 4, FAKE, FAKE, FAKE, 1 << 40, None)
    for kw in (dict(ldo=0), dict(ldo=47), dict(out=FAKE + 4), dict(out=FAKE + 4 * 48), dict(out=FAKE, ldo=96), dict(out=FAKE - 4 * 48 * 3),
               dict(ldy=100, ldo=100, out=FAKE + 4 * 47), dict(ldo=-40)):
        assert call(**kw) == 34, kw


@pytest.mark.gpu
@pytest.mark.parametrize("new,lens", [([1, 2], [900, 70]), ([200, 90], [900, 300])])
def test_attention_out_in_other_places(cuda, new, lens):
    torch = cuda
    from hxq_b200 import serving as S
    c, q, starts, sd, ld, table = _attention_case(torch, S, new, lens, 2, 3, 64, 16, "int8", "bf16")
    want, T = c.attention(q, sd, ld, table, max(new)), q.shape[0]
    same = q.clone()
    assert c.attention(same, sd, ld, table, max(new), out=same).data_ptr() == same.data_ptr() and torch.equal(same, want)
    wide = torch.randn((T, 18, 64), device="cuda").to(torch.bfloat16)   # q and out in one buffer, as projections leave them
    wide[:, 6:12] = q
    for at in (0, 12, 6):
        c.attention(wide[:, 6:12], sd, ld, table, max(new), out=wide[:, at:at + 6])
        assert torch.equal(wide[:, at:at + 6], want)
    heads_first = torch.zeros((6, T, 64), dtype=q.dtype, device="cuda").transpose(0, 1)
    assert torch.equal(c.attention(q, sd, ld, table, max(new), out=heads_first), want)
    row = q[:1].expand(T, -1, -1)   # one row for all
    assert torch.equal(c.attention(row, sd, ld, table, max(new)), c.attention(row.contiguous(), sd, ld, table, max(new)))
    for bad in (q[:1].clone().expand(T, -1, -1), q[:, :1].clone().expand(-1, 6, -1), torch.as_strided(q.clone(), q.shape, (64, 64, 1))):
        with pytest.raises(RuntimeError):
            c.attention(q, sd, ld, table, max(new), out=bad)
    long = torch.randn((T + 1, 6, 64), device="cuda").to(torch.bfloat16)
    with pytest.raises(RuntimeError):
        c.attention(long[:T], sd, ld, table, max(new), out=long[1:])


@pytest.mark.gpu
@pytest.mark.parametrize("O", [48, 50])
def test_lora_out_in_other_places(cuda, O):
    torch = cuda
    from hxq_b200 import serving as S
    i = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    a, b = torch.randn((2, 8, 64), device="cuda").bfloat16(), torch.randn((2, O, 8), device="cuda").bfloat16()
    h, T = S.LoraAdapters(a, b, torch.ones(2, device="cuda")), 90
    x, y = torch.randn((T, 64), device="cuda").bfloat16(), torch.randn((T, O), device="cuda")
    plan = S.lora_plan(i(0, 70, 80, 90), i(0, -1, 1), 2, T)
    want = h.add(y, x, plan)
    both = torch.zeros((T, 2 * O), device="cuda")
    both[:, :O] = y
    assert torch.equal(h.add(both[:, :O], x, plan, out=both[:, O:]), want) and torch.equal(both[:, :O], y)
    assert torch.equal(h.add(both[:, :O], x, plan, out=both[:, :O]), want)
    bias = y[:1].expand(T, -1)
    assert torch.equal(h.add(bias, x, plan), h.add(bias.contiguous(), x, plan))
    long = torch.randn((T + 1, O), device="cuda")
    for yy, out in ((y, y[:1].clone().expand(T, -1)), (long[:T], long[1:]), (both[:, :O], both[:, 4:O + 4])):
        with pytest.raises(RuntimeError):
            h.add(yy, x, plan, out=out)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 9, 70])
@pytest.mark.parametrize("R", [8, 40, 128])
def test_lora_keeps_24_bits(cuda, R, T):
    """x A^T of 24 significant bits by its making, through a B that picks one:
    all of them arrive."""
    torch = cuda
    from hxq_b200 import serving as S
    i = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    g = torch.Generator().manual_seed(R + T)
    I, O = 320, 64
    x, a, b = torch.zeros((T, I)), torch.zeros((1, R, I)), torch.zeros((1, O, R))
    x[:, 3], x[:, 100], x[:, 300] = 1.0, 2.0 ** -8, 2.0 ** -16
    for k in (3, 100, 300):   # 8 bits each: products and their sum are exact
        a[0, :, k] = (torch.randint(128, 256, (R,), generator=g) / 128) * (torch.randint(0, 2, (R,), generator=g) * 2 - 1)
    pick = torch.randint(0, R, (O,), generator=g)
    b[0, torch.arange(O), pick] = 1.0
    h = (x.double() @ a[0].double().T)[:, pick]
    out = S.LoraAdapters(a.bfloat16().cuda(), b.bfloat16().cuda(), torch.ones(1, device="cuda")).add(
        torch.zeros((T, O), device="cuda"), x.bfloat16().cuda(), S.lora_plan(i(0, T), i(0), 1, T))
    # eight additions at most that may truncate, 2^-23 each; without the third part of h 2^-17 and more is lost
    assert bool(((out.double().cpu() - h).abs() <= h.abs() * 2.0 ** -20).all())


@pytest.mark.gpu
@pytest.mark.parametrize("R", [8, 32])
def test_lora_near_the_top_of_fp32(cuda, R):
    """s x A^T between bf16's largest and fp32's: no infinity comes of it."""
    torch = cuda
    from hxq_b200 import serving as S
    i = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    x, a, b = (torch.zeros(n, device="cuda") for n in ((3, 64), (1, R, 64), (1, 16, R)))
    x[:, 7] = torch.tensor([1.0, -1.0, math.inf], device="cuda")
    a[0, :, 7], b[0] = 255 / 128, 2.0 ** -40
    b[0, :, 1:] = 0
    scale = torch.tensor([1.7065e38], device="cuda")
    f = float(scale.double()) * 255 / 128
    assert 3.3962e38 < f < 3.4028e38
    out = S.LoraAdapters(a.bfloat16(), b.bfloat16(), scale).add(torch.zeros((3, 16), device="cuda"), x.bfloat16(), S.lora_plan(i(0, 3), i(0), 1, 3))
    want = f * 2.0 ** -40
    assert bool(((out[0].double() - want).abs() <= want * 2.0 ** -21).all()) and bool(((out[1].double() + want).abs() <= want * 2.0 ** -21).all())
    assert not bool(out[2].isfinite().any())


def test_plan_arrays_that_overlap(H, L):
    """While some CTAs write the plan others still read the lengths."""
    names = ["starts", "lens", "slots", "pos", "taken", "table", "new", "cached", "free"]
    size = dict(new=3, cached=3, table=12, free=5, starts=4, lens=3, slots=8, pos=8, taken=1)
    place = {n: FAKE + 4096 * k for k, n in enumerate(names)}

    def call(**kw):
        d = dict(place, **kw)
        return L.hxq_cuda_kv_plan(d["new"], d["cached"], 3, d["table"], 4, 16, d["free"], 5, d["starts"], d["lens"], d["slots"], d["pos"], 8,
                                  d["taken"], None, None)
    for i, written in enumerate(names[:6]):
        for other in names[i + 1:]:
            assert call(**{written: place[other]}) == 34, (written, other)
            assert call(**{written: place[other] + 4 * size[other] - 4}) == 34, (written, other)
            assert call(**{written: place[other] - 4 * size[written] + 4}) == 34, (written, other)


@pytest.mark.gpu
def test_plan_arrays_side_by_side(H, L, cuda):
    """In one buffer without a gap, as the PyTorch calls lay them out, and the
    lengths read twice."""
    torch = cuda
    buf = torch.zeros(64, dtype=torch.int32, device="cuda")
    at, sizes = {}, dict(new=3, table=6, free=4, starts=4, lens=3, slots=8, pos=8, taken=1)
    k = 0
    for n, size in sizes.items():
        at[n], k = buf[k:k + size], k + size
    at["new"].copy_(torch.tensor([2, 17, 1]))
    at["free"].copy_(torch.tensor([5, 6, 7, 8]))
    p = {n: t.data_ptr() for n, t in at.items()}
    assert L.hxq_cuda_kv_plan(p["new"], p["new"], 3, p["table"], 2, 16, p["free"], 4, p["starts"], p["lens"], p["slots"], p["pos"], 8, p["taken"],
                              None, torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    assert at["starts"].tolist() == [0, 2, 19, 20] and at["lens"].tolist() == [4, 34, 2] and at["pos"].tolist() == [2, 3, 17, 18, 19, 20, 21, 22]


@pytest.mark.gpu
def test_sizes_past_32_bits(cuda):
    """Refused, and not cut to their lower half."""
    torch = cuda
    from hxq_b200 import serving as S
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB")
    N = (1 << 32) + 1
    long = torch.empty(N, dtype=torch.int32, device="cuda")
    i = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    c = S.KvCache.allocate(4, 1, 64)
    rows = torch.ones((1, 1, 64), device="cuda").expand(N, -1, -1)
    q = torch.ones((1, 1, 64), dtype=torch.bfloat16, device="cuda")
    for call in (lambda: c.append(rows, rows, long), lambda: c.read(long), lambda: S.kv_plan(i(1), i(0), long.view(1, -1), i(2), 16, 1),
                 lambda: S.kv_plan(i(1), i(0), i(0).view(1, 1), long, 16, 1), lambda: S.kv_plan(long, long, long.view(-1, 1), i(2), 16, 1),
                 lambda: c.attention(q.expand(N, -1, -1), i(0, 1), i(1), i(0).view(1, 1), 1),
                 lambda: c.attention(q, i(0, 1), i(1), long.view(1, -1), 1)):
        with pytest.raises(ValueError, match="2\\^31"):
            call()
    assert bool((c.k == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_of_prompts_replayed_with_other_lengths(cuda, dim):
    """Two graphs over the kernel for many rows, replayed at once."""
    torch = cuda
    from hxq_b200 import serving as S
    lens = [900, 130, 2000]
    c, q, _, _, ld, table = _attention_case(torch, S, [300, 130, 80], lens, 2, 2, dim, 16, "e4m3", "bf16")
    sd = torch.tensor([0, 300, 430, 510], dtype=torch.int32, device="cuda")
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c.attention(q, sd, ld, table, 300)
    graphs = []
    for _ in range(2):
        g, out = torch.cuda.CUDAGraph(), torch.full_like(q, 9.0)
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        with torch.cuda.graph(g, stream=side):
            c.attention(q, sd, ld, table, 300, window=700, out=out, status=status)
        graphs.append((g, out, status))
    for new in ([300, 130, 80], [1, 2, 500], [0, 130, 1], [64, 65, 0], [300, 130, 80]):
        starts = [0, new[0], new[0] + new[1], sum(new)]
        sd.copy_(torch.tensor(starts, dtype=torch.int32))
        torch.cuda.synchronize()
        with torch.cuda.stream(other):
            graphs[0][0].replay()
        graphs[1][0].replay()
        torch.cuda.synchronize()
        want, _, tol, _ = _attention_ref(torch, c, q, starts, lens, table, dim ** -0.5, 700, True)
        n = starts[-1]
        for _, out, status in graphs:
            assert int(status) == 0 and bool(((out[:n].double() - want[:n]).abs() <= tol[:n]).all()), new
        assert torch.equal(graphs[0][1][:n], graphs[1][1][:n])


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 140])
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_value_scales_far_apart(cuda, new, dim):
    """Values of 0 and of 2^40 times a code, seen with the same weight: those of
    0 count in the softmax's sum."""
    torch = cuda
    from hxq_b200 import serving as S
    n, P = 320, 16
    c = S.KvCache.allocate(n // P, 1, dim, P)
    i = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    c.v.fill_(64)
    c.v_scales.copy_(torch.where(torch.arange(n // P, device="cuda") % 2 == 0, 0.0, 2.0 ** 40)[:, None])
    q, lse = torch.ones((new, 2, dim), dtype=torch.bfloat16, device="cuda"), torch.zeros((new, 2), device="cuda")
    o = c.attention(q, i([0, new]), i([n]), torch.arange(n // P, dtype=torch.int32, device="cuda").view(1, -1), new, causal=False, lse=lse)
    # half of the keys: exact in f16 and fp32 but for the inverses of the scales and the sum (2^-20), and out in bf16
    assert bool(((o.double() / 2.0 ** 45 - 1).abs() <= 2.0 ** -8).all())
    assert bool(((lse.double() - math.log(n)).abs() <= 2.0 ** -19 * math.log(n)).all())
