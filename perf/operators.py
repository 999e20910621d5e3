"""Cases of the serving operators: step plans, the 8-bit KV cache, attention
over it, and low-rank adapters beside a shared projection.

Each case is one call (or one call and its read-back) of a serving step on a
model of the 7B shape (4096 / 11008 features, heads of 128) or on a generic
grouped-query one.  `run` computes the plain form with elementary torch
operations in 32 bits, or calls the framework's operators where `own` is set.
"""
import math
import random
import sys

import torch

own = False

QMAX = {"int8": 127.0, "e4m3": 448.0}
CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _serving():
    if "hxq-native_b200" not in sys.path:
        sys.path.insert(1, "hxq-native_b200")
    from hxq_b200 import serving
    return serving


# -- cases -------------------------------------------------------------------

def listed():
    return [
        # one decode step of 64 requests: every request adds one token
        dict(name="plan_decode", op="plan", batch=64, new=1, cached=4096, block=16, shape=1),
        # a large admission: prompts of up to 1024 tokens, some with a cached prefix
        dict(name="plan_prompts", op="plan", batch=500, new=1024, cached=1500, block=32, shape=2),
        # the step's keys and values of 64 decoding requests, and their blocks read back
        dict(name="append_decode", op="append", batch=64, new=1, cached=2000, heads=8, dim=128, block=16,
             format="int8", type="bf16", shape=3),
        # prompts written into fresh and half-filled blocks, 32 heads
        dict(name="append_prompts", op="append", batch=9, new=2048, cached=100, heads=32, dim=128, block=64,
             format="e4m3", type="bf16", shape=4),
        # one request, one token, a short context: the latency of a call
        dict(name="attention_one", op="attention", batch=1, new=1, cached=1023, heads=32, group=1, dim=128, block=16,
             format="int8", type="bf16", window=0, even=True, shape=5),
        # a decode step of a ragged batch, grouped heads
        dict(name="attention_decode", op="attention", batch=64, new=1, cached=8191, heads=8, group=4, dim=128, block=16,
             format="int8", type="bf16", window=0, even=False, shape=6),
        # two long documents: few rows, a long axis
        dict(name="attention_long", op="attention", batch=2, new=1, cached=131000, heads=8, group=4, dim=128, block=64,
             format="e4m3", type="f16", window=0, even=True, shape=7),
        # whole prompts
        dict(name="attention_prompts", op="attention", batch=3, new=4096, cached=0, heads=32, group=1, dim=128, block=16,
             format="int8", type="bf16", window=0, even=False, shape=8),
        # a chunk of a long prompt over what is held already, sliding window, heads of 64
        dict(name="attention_chunk", op="attention", batch=2, new=512, cached=16000, heads=8, group=5, dim=64, block=32,
             format="e4m3", type="bf16", window=4096, even=True, shape=9),
        # 64 decoding requests over 16 adapters, an attention projection
        dict(name="lora_decode", op="lora", batch=64, new=1, adapters=16, rank=16, inf=4096, outf=4096, shape=10),
        # a mixed step: decoding requests and short prompts, the up projection
        dict(name="lora_mixed", op="lora", batch=40, new=50, adapters=24, rank=64, inf=4096, outf=11008, shape=11),
        # long prompts of few adapters, the down projection
        dict(name="lora_prompts", op="lora", batch=6, new=2048, adapters=4, rank=32, inf=11008, outf=4096, shape=12),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["plan", "append", "attention", "attention", "lora", "lora"])
    shape = rng.randrange(1, 1 << 30)
    if op == "plan":
        return dict(op=op, batch=_log(rng, 1, 1000), new=_log(rng, 1, 1024), cached=_log(rng, 1, 8192),
                    block=rng.choice([16, 32, 64, 128]), shape=shape)
    if op == "append":
        heads, new = rng.choice([1, 4, 8, 32]), _log(rng, 1, 2048)
        return dict(op=op, batch=_log(rng, 1, max(1, min(128, 16384 // new))), new=new, cached=_log(rng, 1, 2000), heads=heads,
                    dim=rng.choice([64, 128, 256]), block=rng.choice([16, 32, 64, 128]),
                    format=rng.choice(["int8", "e4m3"]), type=rng.choice(["bf16", "f16", "f32"]), shape=shape)
    if op == "attention":
        heads, group, dim = rng.choice([1, 2, 4, 8, 32]), rng.choice([1, 2, 4, 5, 7, 8, 16]), rng.choice([64, 128])
        heads = min(heads, 64 // group)
        if rng.random() < 0.6:
            new, cached = rng.choice([1, 1, 1, 2, 4]), _log(rng, 1, 65536)
            most = max(1, 300_000_000 // ((cached + new) * heads * dim))
            batch = _log(rng, 1, min(128, most))
        else:
            new, cached = _log(rng, 16, 2048), rng.choice([0, 0, _log(rng, 1, 8192)])
            most = max(1, 800_000_000 // (new * (cached + new) * heads * group))
            batch = _log(rng, 1, min(8, most))
        return dict(op=op, batch=batch, new=new, cached=cached, heads=heads, group=group, dim=dim,
                    block=rng.choice([16, 32, 64, 128]), format=rng.choice(["int8", "e4m3"]),
                    type=rng.choice(["bf16", "f16"]), window=rng.choice([0, 0, 0, _log(rng, 1, 4096)]),
                    even=rng.random() < 0.3, shape=shape)
    new = rng.choice([1, 1, _log(rng, 1, 2048)])
    return dict(op=op, batch=_log(rng, 1, max(1, min(256, 8192 // new))), new=new, adapters=_log(rng, 1, 32),
                rank=rng.choice([8, 16, 32, 64, 128]), inf=64 * _log(rng, 4, 172), outf=8 * _log(rng, 32, 1376), shape=shape)


def _lengths(case):
    """New and held tokens of each request: the listed number for every
    request where the case is even or the number is one, otherwise up to it,
    the first request with the most."""
    rng, B = random.Random(case["shape"]), case["batch"]
    even = case.get("even", False)
    new = [case["new"] if even or b == 0 or case["new"] == 1 else rng.randint(1, case["new"]) for b in range(B)]
    cached = [case["cached"] if even or b == 0 else rng.randint(0, case["cached"]) for b in range(B)]
    return new, cached


def _requests(case):
    """Tokens and adapter (-1: none) of each request of an adapter case."""
    rng, B = random.Random(case["shape"]), case["batch"]
    new = [case["new"] if b == 0 or case["new"] == 1 else rng.randint(1, case["new"]) for b in range(B)]
    ids = [rng.randrange(case["adapters"]) if b == 0 or rng.random() < 0.9 else -1 for b in range(B)]
    return new, ids


def _pairs(n, c, window):
    """Query-key pairs of one request."""
    if not window:
        return n * c + n * (n + 1) // 2
    return sum(min(window, c + i + 1) for i in range(n))


def work(case):
    op = case["op"]
    if op == "lora":
        new, ids = _requests(case)
        T, used, live = sum(new), len({i for i in ids if i >= 0}), sum(n for n, i in zip(new, ids) if i >= 0)
        r, i, o = case["rank"], case["inf"], case["outf"]
        return {"bytes": live * i * 2 + T * o * 8 + used * r * (i + o) * 2, "flops": 2 * live * r * (i + o)}
    new, cached = _lengths(case)
    T, P = sum(new), case["block"]
    if op == "plan":
        fresh = sum(-(-(n + c) // P) - -(-c // P) for n, c in zip(new, cached))
        return {"bytes": 16 * case["batch"] + 8 * T + 8 * fresh, "flops": 0}
    H, D = case["heads"], case["dim"]
    if op == "append":
        size = 4 if case["type"] == "f32" else 2
        back = sum(n + c % P for n, c in zip(new, cached))
        return {"bytes": 2 * H * D * (T * (size + 1) + back * 3), "flops": 0}
    w = case["window"]
    pairs = sum(_pairs(n, c, w) for n, c in zip(new, cached))
    keys = sum(min(n + c, w + n - 1) if w else n + c for n, c in zip(new, cached))
    return {"bytes": 2 * H * D * (keys + T * case["group"] * 2), "flops": 4 * D * H * case["group"] * pairs}


# -- inputs ------------------------------------------------------------------

def _ints(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def _pages(cached, new, P, n_blocks, gen, dev):
    """A block table over shuffled blocks for requests of cached + new tokens,
    and the blocks that are left."""
    counts = [-(-(c + n) // P) for c, n in zip(cached, new)]
    order = torch.randperm(n_blocks, generator=gen, device=dev).to(torch.int32)
    W, off = max(counts), torch.tensor([sum(counts[:b]) for b in range(len(counts))], device=dev)
    j = torch.arange(W, device=dev)
    at = torch.clamp(off[:, None] + j[None, :], max=n_blocks - 1)
    table = torch.where(j[None, :] < torch.tensor(counts, device=dev)[:, None], order[at], 0)
    return table.to(torch.int32).contiguous(), order[sum(counts):]


def _fill(shape, fmt, gen, dev):
    """Codes as a cache of near-normal vectors holds them, and scales."""
    codes = torch.empty(shape, dtype=CODES[fmt], device=dev)
    flat, step = codes.view(shape[0], -1), max(1, (1 << 26) // max(1, math.prod(shape[1:])))
    for at in range(0, shape[0], step):
        x = torch.randn(flat[at:at + step].shape, generator=gen, device=dev).clamp_(-3.5, 3.5) * (QMAX[fmt] / 3.5)
        flat[at:at + step] = (x.round() if fmt == "int8" else x).to(CODES[fmt])
    scales = torch.exp(0.5 * torch.randn(shape[:2], generator=gen, device=dev)) * (3.5 / QMAX[fmt])
    return codes, scales


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    s = dict(case)
    if case["op"] == "lora":
        new, ids = _requests(case)
        T, r, n = sum(new), case["rank"], case["adapters"]
        s["starts"] = _ints([sum(new[:b]) for b in range(len(new) + 1)], dev)
        s["ids"] = _ints(ids, dev)
        s["x"] = torch.randn((T, case["inf"]), generator=gen, device=dev).to(torch.bfloat16)
        s["y"] = torch.randn((T, case["outf"]), generator=gen, device=dev)
        s["a"] = (torch.randn((n, r, case["inf"]), generator=gen, device=dev) / math.sqrt(case["inf"])).to(torch.bfloat16)
        s["b"] = (torch.randn((n, case["outf"], r), generator=gen, device=dev) * 0.1).to(torch.bfloat16)
        s["scales"] = torch.rand((n,), generator=gen, device=dev) + 0.5
        if own:
            s["adapters_handle"] = _serving().LoraAdapters(s["a"], s["b"], s["scales"])
        return s
    new, cached = _lengths(case)
    T, P = sum(new), case["block"]
    need = sum(-(-(c + n) // P) for c, n in zip(cached, new))
    n_blocks = need + need // 8 + 8
    s["table"], rest = _pages(cached, new, P, n_blocks, gen, dev)
    s["starts"] = _ints([sum(new[:b]) for b in range(len(new) + 1)], dev)
    s["new_lens"], s["cached_lens"] = _ints(new, dev), _ints(cached, dev)
    s["lens"], s["T"] = s["new_lens"] + s["cached_lens"], T
    if case["op"] == "plan":
        held = torch.tensor([-(-c // P) for c in cached], device=dev)
        j = torch.arange(s["table"].shape[1], device=dev)
        lost = (j[None, :] >= held[:, None]) & (j[None, :] < torch.tensor([-(-(c + n) // P) for c, n in zip(cached, new)], device=dev)[:, None])
        s["free"] = torch.cat([s["table"][lost], rest]).contiguous()  # what the step takes comes from the free list
        s["table"] = torch.where(lost, -1, s["table"])
        return s
    H, D, fmt = case["heads"], case["dim"], case["format"]
    s["k"], s["k_scales"] = _fill((n_blocks, H, P, D), fmt, gen, dev)
    s["v"], s["v_scales"] = _fill((n_blocks, H, P, D), fmt, gen, dev)
    if own:
        s["cache"] = _serving().KvCache(s["k"], s["v"], s["k_scales"], s["v_scales"])
    if case["op"] == "attention":
        s["q"] = torch.randn((T, H * case["group"], D), generator=gen, device=dev).to(TYPES[case["type"]])
        s["max_new"], s["max_len"] = max(new), max(n + c for n, c in zip(new, cached))
        return s
    dtype = TYPES[case["type"]]
    s["new_k"] = (1.2 * torch.randn((T, H, D), generator=gen, device=dev)).to(dtype)
    s["new_v"] = (1.2 * torch.randn((T, H, D), generator=gen, device=dev)).to(dtype)
    pos = [c + i for n, c in zip(new, cached) for i in range(n)]
    req = [b for b, n in enumerate(new) for _ in range(n)]
    t, p = torch.tensor(req, device=dev), torch.tensor(pos, device=dev)
    blocks = s["table"][t, p // P]
    s["slots"] = (blocks * P + p % P).to(torch.int32)
    # what the block manager knows of the step: the blocks it touches, and which of them each token is in
    seen = {}
    s["touch"] = torch.tensor([seen.setdefault((b, q // P), len(seen)) for b, q in zip(req, pos)], device=dev)
    where = torch.tensor(list(seen), device=dev)
    s["blocks"] = s["table"][where[:, 0], where[:, 1]].long()
    back = [(b, q) for b, (n, c) in enumerate(zip(new, cached)) for q in range(c - c % P, c + n)]
    back = torch.tensor(back, device=dev)
    s["back"] = (s["table"][back[:, 0], back[:, 1] // P] * P + back[:, 1] % P).to(torch.int32)
    return s


# -- plain forms ---------------------------------------------------------------

def _plan(s):
    P, T, dev = s["block"], s["T"], s["table"].device
    new, cached, table, free = s["new_lens"].long(), s["cached_lens"].long(), s["table"].clone(), s["free"]
    lens = new + cached
    starts = torch.cat([torch.zeros(1, dtype=torch.int64, device=dev), torch.cumsum(new, 0)])
    held, total = (cached + P - 1) // P, (lens + P - 1) // P
    need = total - held
    base = torch.cumsum(need, 0) - need
    j = torch.arange(table.shape[1], device=dev)[None, :]
    at = base[:, None] + j - held[:, None]
    fresh = (j >= held[:, None]) & (j < total[:, None])
    table = torch.where(fresh, torch.where(at < free.numel(), free[at.clamp(0, free.numel() - 1)], -1), table)
    t = torch.arange(T, device=dev)
    b = torch.searchsorted(starts, t, right=True) - 1
    pos = cached[b] + t - starts[b]
    block = table[b, pos // P]
    slots = torch.where(block >= 0, block * P + pos % P, -1)
    return [starts.int(), lens.int(), table.int(), slots.int(), pos.int(), need.sum().clamp(max=free.numel()).int().reshape(1)]


def _append_one(codes, scales, x, s, fmt):
    P, q = s["block"], QMAX[fmt]
    n, H = s["blocks"].numel(), x.shape[1]
    pos = s["slots"].long() % P
    x = x.float()
    most = torch.zeros((n, H), device=x.device).index_reduce_(0, s["touch"], x.abs().amax(-1), "amax")
    fresh = torch.zeros(n, dtype=torch.int32, device=x.device).index_add_(0, s["touch"], (pos == 0).int()) > 0
    old = torch.where(fresh[:, None], 0.0, scales[s["blocks"]])
    scale = torch.maximum(old, most / q)
    scale = torch.where(scale < 2.0 ** -126, 0.0, scale)
    inv = torch.where(scale > 0, 1.0 / scale, 0.0)
    held = codes[s["blocks"]].float()
    ratio = torch.where(scale > 0, old / scale, 0.0)
    moved = held * ratio[:, :, None, None]
    fit = (lambda v: v.round().clamp(-q, q).to(torch.int8)) if fmt == "int8" else (lambda v: v.clamp(-q, q).to(torch.float8_e4m3fn))
    grown = ((scale > old) & ~fresh[:, None])[:, :, None, None]
    body = torch.where(grown, fit(moved).float(), held)
    body[s["touch"], :, pos] = fit(x * inv[s["touch"]][:, :, None]).float()
    codes.view(torch.int8)[s["blocks"]] = body.to(codes.dtype).view(torch.int8)
    scales[s["blocks"]] = scale


def _read(codes, scales, slots, P):
    at = slots.long()
    return (codes[at // P, :, at % P].float() * scales[at // P][:, :, None]).to(torch.bfloat16)


def _attention(s):
    P, G, D, H, L, Q = s["block"], s["group"], s["dim"], s["heads"], s["max_len"], s["max_new"]
    B, dev = s["lens"].numel(), s["q"].device
    table = s["table"].long()
    k = (s["k"][table].float() * s["k_scales"][table][..., None, None]).transpose(1, 2).reshape(B, H, -1, D)[:, :, :L]
    v = (s["v"][table].float() * s["v_scales"][table][..., None, None]).transpose(1, 2).reshape(B, H, -1, D)[:, :, :L]
    starts, new, lens = s["starts"].long(), s["new_lens"].long(), s["lens"].long()
    i = torch.arange(Q, device=dev)
    at = (starts[:-1, None] + i).clamp(max=s["T"] - 1)
    q = s["q"][at].float().reshape(B, Q, H, G, D).permute(0, 2, 3, 1, 4).reshape(B, H, G * Q, D)
    scores = torch.matmul(q, k.transpose(2, 3)).reshape(B, H, G, Q, L) * (D ** -0.5)
    own_pos = (lens - new)[:, None] + i
    j = torch.arange(L, device=dev)
    seen = j[None, None, :] <= own_pos[:, :, None]
    if s["window"]:
        seen = seen & (j[None, None, :] > own_pos[:, :, None] - s["window"])
    seen = seen & (j[None, None, :] < lens[:, None, None])
    scores = scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp_(scores.sub_(top))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.reshape(B, H, G * Q, L), v).reshape(B, H, G, Q, D) / total
    t = torch.arange(s["T"], device=dev)
    b = torch.searchsorted(starts, t, right=True) - 1
    return o.permute(0, 3, 1, 2, 4).reshape(B, Q, H * G, D)[b, t - starts[b]].to(s["q"].dtype)


def _lora(s):
    T, r, n = s["x"].shape[0], s["rank"], s["adapters"]
    t = torch.arange(T, device=s["x"].device)
    ids = s["ids"].long()[torch.searchsorted(s["starts"].long(), t, right=True) - 1]
    mine = (ids[:, None] == torch.arange(n, device=t.device)[None, :]).float() * s["scales"]
    h = torch.matmul(s["x"].float(), s["a"].float().reshape(n * r, -1).t()).reshape(T, n, r) * mine[:, :, None]
    return s["y"] + torch.matmul(h.reshape(T, n * r), s["b"].float().permute(0, 2, 1).reshape(n * r, -1))


def run(s):
    if own:
        return _own(s)
    if s["op"] == "plan":
        return _plan(s)
    if s["op"] == "append":
        _append_one(s["k"], s["k_scales"], s["new_k"], s, s["format"])
        _append_one(s["v"], s["v_scales"], s["new_v"], s, s["format"])
        return [_read(s["k"], s["k_scales"], s["back"], s["block"]), _read(s["v"], s["v_scales"], s["back"], s["block"]),
                s["k_scales"], s["v_scales"]]
    return [_attention(s) if s["op"] == "attention" else _lora(s)]


def _own(s):
    S = _serving()
    if s["op"] == "plan":
        p = S.kv_plan(s["new_lens"], s["cached_lens"], s["table"], s["free"], s["block"], s["T"])
        return [p.starts, p.lens, s["table"], p.slots, p.positions, p.taken]
    if s["op"] == "append":
        s["cache"].append(s["new_k"], s["new_v"], s["slots"])
        k, v = s["cache"].read(s["back"], torch.bfloat16)
        return [k, v, s["cache"].k_scales, s["cache"].v_scales]
    if s["op"] == "attention":
        return [s["cache"].attention(s["q"], s["starts"], s["lens"], s["table"], max_new=s["max_new"], window=s["window"])]
    plan = S.lora_plan(s["starts"], s["ids"], s["adapters"], s["x"].shape[0])
    return [s["adapters_handle"].add(s["y"], s["x"], plan)]


# -- the definition in 64 bits -------------------------------------------------

def exact(case, seed):
    if case["op"] == "plan":
        return None
    s = prepare(case, seed)
    if case["op"] == "lora":
        out = s["y"].double()
        at, ids = s["starts"].tolist(), s["ids"].tolist()
        for b, a in enumerate(ids):
            if a >= 0:
                rows = slice(at[b], at[b + 1])
                out[rows] += s["scales"][a].double() * (s["x"][rows].double() @ s["a"][a].double().T @ s["b"][a].double().T)
        return [out]
    P = case["block"]
    if case["op"] == "append":
        q, got = QMAX[case["format"]], []
        scales_out = []
        for codes, scales, x in ((s["k"], s["k_scales"], s["new_k"]), (s["v"], s["v_scales"], s["new_v"])):
            values = codes.double() * scales.double()[:, :, None, None]
            scales = scales.double()
            x = x.double()
            slots = s["slots"].long()
            for page in s["blocks"].tolist():
                mine = (slots // P == page).nonzero()[:, 0]
                pos = slots[mine] % P
                old = torch.zeros_like(scales[page]) if bool((pos == 0).any()) else scales[page]
                scale = torch.maximum(old, x[mine].abs().amax(-1).amax(0) / q)
                grown = scale > old
                body = values[page] / scale[:, None, None]
                body = torch.where(grown[:, None, None], _fit64(body, case["format"]), body)
                body[:, pos] = _fit64(x[mine] / scale[None, :, None], case["format"]).transpose(0, 1)
                values[page], scales[page] = body * scale[:, None, None], scale
            at = s["back"].long()
            got.append(values[at // P, :, at % P])
            scales_out.append(scales)
        return got + scales_out
    G, D, H, w = case["group"], case["dim"], case["heads"], case["window"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    at, lens = s["starts"].tolist(), s["lens"].tolist()
    if sum((at[b + 1] - at[b]) * n for b, n in enumerate(lens)) * H * G * D > 1 << 40:
        return None
    for b, n in enumerate(lens):
        pages = s["table"][b, :-(-n // P)].long()
        rows, length = slice(at[b], at[b + 1]), at[b + 1] - at[b]
        p = torch.arange(n - length, n, device=out.device)
        j = torch.arange(n, device=out.device)
        mask = (j[None, :] > p[:, None]) | ((j[None, :] <= p[:, None] - w) if w else torch.zeros_like(j[None, :], dtype=torch.bool))
        for h in range(H):
            k = (s["k"][pages, h].double() * s["k_scales"][pages, h].double()[:, None, None]).reshape(-1, D)[:n]
            v = (s["v"][pages, h].double() * s["v_scales"][pages, h].double()[:, None, None]).reshape(-1, D)[:n]
            for g in range(G):
                scores = (s["q"][rows, h * G + g].double() @ k.T / math.sqrt(D)).masked_fill(mask, -math.inf)
                out[rows, h * G + g] = torch.softmax(scores, -1) @ v
    return [out]


def _fit64(x, fmt):
    """Nearest code, as a value."""
    if fmt == "int8":
        return x.round().clamp(-127, 127)
    x = x.clamp(-448, 448)
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step
