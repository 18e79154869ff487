"""The operators of the 4-bit (MXFP4) paged cache as measured cases: block tables and slot maps
from request lengths, the cache's write, decode attention over it, prefill attention over it.

A cache is a uint8 tensor (num_pages, kv_heads, 17 * head_dim): for one kv head of a 16-token
page the K codes, the V codes and their scales. Codes are E2M1 (two per byte, the even dim in
the low nibble), scales E8M0, one per 32 dims of a row:
  K code byte of (token t, dim d)   t * D/2 + d/2
  V code byte                       8 D + (d/W) 8 W + (t/4) 2 W + (d%W / (W/16)) W/8
                                      + (t%4) W/32 + (d % (W/16)) / 2,      W = min(D, 128)
  K scale byte of block b           16 D + 16 b + t,    V scale byte: D/2 further
"""
import math
import random

import torch

own = False

DEV = "cuda"
PAGE = 16
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------- cases

def listed():
    return [
        # one decode step of a serving batch: every request gets one more token
        dict(name="tables_step", op="tables", batch=32, cached_lo=1, cached_hi=8192, new_lo=1,
             new_hi=1, blocks=1024),
        # a prefill batch of unequal chunks behind unequal prefixes
        dict(name="tables_prefill", op="tables", batch=8, cached_lo=0, cached_hi=500, new_lo=33,
             new_hi=777, blocks=128),
        # a large mixed step: long prefixes, up to 64 new tokens each
        dict(name="tables_mixed", op="tables", batch=500, cached_lo=0, cached_hi=4001, new_lo=1,
             new_hi=64, blocks=512),
        # the decode step's cache write of 32 requests
        dict(name="write_step", op="write", tokens=32, pad=0, hq=32, hkv=8, d=64, dtype="bf16",
             style=0, far=2048),
        # a prefill chunk's cache write
        dict(name="write_prefill", op="write", tokens=8192, pad=0, hq=32, hkv=8, d=128,
             dtype="bf16", style=0, far=131072),
        # wide heads, interleaved pairs, a batch padded behind its last token
        dict(name="write_odd", op="write", tokens=777, pad=23, hq=16, hkv=4, d=256, dtype="fp16",
             style=1, far=8192),
        # two short requests, where latency counts
        dict(name="decode_small", op="decode", batch=2, lo=512, hi=512, hq=32, hkv=8, d=128,
             dtype="fp16", window=0, cap=0.0, sinks=False),
        # a serving batch of long contexts
        dict(name="decode_batch", op="decode", batch=32, lo=8192, hi=8192, hq=32, hkv=8, d=128,
             dtype="fp16", window=0, cap=0.0, sinks=False),
        # unequal lengths, narrow heads, attention sinks
        dict(name="decode_ragged", op="decode", batch=128, lo=128, hi=8192, hq=64, hkv=8, d=64,
             dtype="bf16", window=0, cap=0.0, sinks=True),
        # one very long context, 16 q heads per kv head
        dict(name="decode_long", op="decode", batch=1, lo=131071, hi=131071, hq=128, hkv=8, d=128,
             dtype="bf16", window=0, cap=0.0, sinks=False),
        # prefill of unequal requests behind short prefixes
        dict(name="extend_batch", op="extend", batch=8, prefix_lo=0, prefix_hi=500, new_lo=33,
             new_hi=777, hq=32, hkv=8, d=64, dtype="bf16", window=0, cap=0.0),
        # a chunk of a long prompt over its cached prefix
        dict(name="extend_chunk", op="extend", batch=1, prefix_lo=6144, prefix_hi=6144,
             new_lo=2048, new_hi=2048, hq=32, hkv=8, d=128, dtype="fp16", window=0, cap=0.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["tables", "write", "decode", "extend"])
    dtype = rng.choice(["fp16", "bf16"])
    d = rng.choice([64, 128, 256])
    hkv, group = rng.choice([(1, 8), (2, 4), (4, 4), (8, 1), (8, 4), (8, 5), (8, 8), (3, 7)])
    if op == "tables":
        hi = _log(rng, 20, 8000)
        new = _log(rng, 1, 700)
        return dict(op=op, batch=_log(rng, 1, 500), cached_lo=rng.randrange(0, hi), cached_hi=hi,
                    new_lo=rng.randrange(0, new + 1), new_hi=new, blocks=1024)
    if op == "write":
        return dict(op=op, tokens=_log(rng, 1, 4000), pad=rng.choice([0, 0, 1, 17]),
                    hq=hkv * group, hkv=hkv, d=d, dtype=dtype, style=rng.choice([0, 1]),
                    far=_log(rng, 100, 131072))
    if op == "decode":
        batch = _log(rng, 1, 100)
        hi = _log(rng, 17, min(131072, (1 << 27) // (hkv * d * batch)))
        return dict(op=op, batch=batch, lo=rng.choice([hi, max(1, hi // 10)]), hi=hi,
                    hq=hkv * group, hkv=hkv, d=d, dtype=dtype,
                    window=rng.choice([0, 0, 0, 128, 1000]), cap=rng.choice([0.0, 0.0, 30.0]),
                    sinks=rng.choice([False, False, True]))
    batch = rng.choice([1, 1, 2, 3, 5])
    new = _log(rng, 1, 1500 // batch)
    pre = _log(rng, 1, 6000 // batch)
    return dict(op=op, batch=batch, prefix_lo=rng.randrange(0, pre), prefix_hi=pre,
                new_lo=max(1, new // 2), new_hi=new, hq=hkv * group, hkv=hkv, d=d, dtype=dtype,
                window=rng.choice([0, 0, 500]), cap=rng.choice([0.0, 0.0, 30.0]))


def _spread(lo, hi, n):
    """n lengths evenly over [lo, hi]."""
    return [lo + int((hi - lo) * (i + 0.5) / n) for i in range(n)]


def _pairs(lo, hi, new_lo, new_hi, n):
    """n (tokens before, new tokens), each evenly over its range, paired the same for every seed."""
    new = _spread(new_lo, new_hi, n)
    random.Random(1).shuffle(new)
    return list(zip(_spread(lo, hi, n), new))


def _table_pairs(case):
    most = case["blocks"] * PAGE
    return [(min(c, most - n), n) for c, n in
            _pairs(case["cached_lo"], case["cached_hi"], case["new_lo"], case["new_hi"],
                   case["batch"])]


def _pages(n):
    return -(-n // PAGE)


# ---------------------------------------------------------------- inputs

def _pack(k, v, d):
    """(pages, kv_heads, 17 d) uint8 of fp32 K and V (pages, kv_heads, 16, d)."""
    n, h = k.shape[:2]
    kc, ks = _quantize(k)
    vc, vs = _quantize(v)
    w = min(d, 128)
    kb = (kc[..., 0::2] | kc[..., 1::2] << 4).reshape(n, h, 8 * d)
    vb = vc[..., 0::2] | vc[..., 1::2] << 4                                # (n, h, 16, d/2)
    vb = vb.view(n, h, 4, 4, d // w, 16, w // 32).permute(0, 1, 4, 2, 5, 3, 6)
    return torch.cat([kb, vb.reshape(n, h, 8 * d), ks.transpose(2, 3).reshape(n, h, d // 2),
                      vs.transpose(2, 3).reshape(n, h, d // 2)], dim=2).contiguous()


def _quantize(x):
    """E2M1 codes and E8M0 scale bytes (both uint8) of x's last dim in blocks of 32."""
    b = x.reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    bits = b.abs().amax(-1).float().contiguous().view(torch.int32)
    e = ((bits + (1 << 21)) >> 23) - 2                       # 1.75 and above: the next power
    e = e.clamp(1, 252)
    y = torch.ldexp(b, (127 - e).unsqueeze(-1))
    a = y.abs()
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) +
            (a >= 3.5) + (a > 5.0))
    code = torch.where(y < 0, code + 8, code)
    return code.reshape(x.shape).to(torch.uint8), e.to(torch.uint8)


def _cache(g, pages, hkv, d):
    """A filled pool: unit normal V, K with a few strong channels, as after the projections."""
    cache = torch.empty(pages, hkv, 17 * d, dtype=torch.uint8, device=DEV)
    gain = torch.exp(torch.randn(hkv, 1, d, generator=g, device=DEV) * 0.5)
    gain = gain / gain.square().mean(-1, keepdim=True).sqrt()
    step = max(1, (1 << 25) // (hkv * PAGE * d))
    for i in range(0, pages, step):
        n = min(step, pages - i)
        k = torch.randn(n, hkv, PAGE, d, generator=g, device=DEV) * gain
        v = torch.randn(n, hkv, PAGE, d, generator=g, device=DEV)
        cache[i:i + n] = _pack(k, v, d)
    return cache


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    order = random.Random(seed)
    s = dict(case)
    op = case["op"]
    ints = lambda v, t=torch.int32: torch.tensor(v, dtype=t, device=DEV)  # noqa: E731
    if op == "tables":
        b, blocks = case["batch"], case["blocks"]
        pairs = _table_pairs(case)
        order.shuffle(pairs)
        cached, new = zip(*pairs)
        need = sum(_pages(c + n) - _pages(c) for c, n in zip(cached, new))
        ids = torch.randperm(b * blocks + need, generator=g, device=DEV).to(torch.int32)
        rows = torch.randperm(2 * b, generator=g, device=DEV)[:b]
        table = torch.full((2 * b, blocks), -1, dtype=torch.int32, device=DEV)
        table[rows] = ids[:b * blocks].view(b, blocks)
        live = torch.arange(blocks, device=DEV) < ints([_pages(c) for c in cached])[:, None]
        table[rows] = torch.where(live, table[rows], ints(-1))
        s.update(table=table, rows=rows, cached=ints(cached, torch.int64),
                 new=ints(new, torch.int64), new_pages=ids[b * blocks:].clone(),
                 num_tokens=sum(new), capacity=sum(_pages(c + n) for c, n in zip(cached, new)))
        return s
    dt = DTYPES[case["dtype"]]
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    if op == "write":
        t = case["tokens"] + case["pad"]
        pages = _pages(case["tokens"]) + 8
        kv = torch.randn(t, 2, hkv, d, generator=g, device=DEV).to(dt)
        slots = torch.full((t,), -1, dtype=torch.int32, device=DEV)
        ids = torch.randperm(pages, generator=g, device=DEV)[:_pages(case["tokens"])]
        at = ids[:, None] * PAGE + torch.arange(PAGE, device=DEV)
        slots[:case["tokens"]] = at.reshape(-1)[:case["tokens"]].to(torch.int32)
        start = int(torch.randint(0, max(1, case["far"] - t), (1,), generator=g, device=DEV))
        i = torch.arange(0, d, 2, dtype=torch.float64, device=DEV)
        s.update(q=torch.randn(t, hq, d, generator=g, device=DEV).to(dt), k=kv[:, 0], v=kv[:, 1],
                 slots=slots, positions=torch.arange(start, start + t, device=DEV).to(torch.int32),
                 inv_freq=(500000.0 ** (-i / d)).float(),
                 cache=torch.zeros(pages, hkv, 17 * d, dtype=torch.uint8, device=DEV))
        return s
    if op == "decode":
        b = case["batch"]
        lens = _spread(case["lo"], case["hi"], b)
        order.shuffle(lens)
        np_ = [_pages(n) for n in lens]
        total = sum(np_)
        s.update(q=torch.randn(b, hq, d, generator=g, device=DEV).to(dt),
                 cache=_cache(g, total + 3, hkv, d),
                 indptr=ints([sum(np_[:i]) for i in range(b + 1)]),
                 indices=torch.randperm(total + 3, generator=g, device=DEV)[:total].to(torch.int32),
                 last=ints([n - PAGE * (p - 1) for n, p in zip(lens, np_)]), hint=max(np_),
                 sink=torch.randn(hq, generator=g, device=DEV) if case["sinks"] else None)
        return s
    b = case["batch"]
    pairs = _pairs(case["prefix_lo"], case["prefix_hi"], case["new_lo"], case["new_hi"], b)
    order.shuffle(pairs)
    new, alls = [n for _, n in pairs], [p + n for p, n in pairs]
    width = max(_pages(n) for n in alls)
    pages = sum(_pages(n) for n in alls)
    ids = torch.randperm(pages + 2, generator=g, device=DEV).to(torch.int32)
    table = torch.full((b + 1, width), -1, dtype=torch.int32, device=DEV)
    at = 0
    for i, n in enumerate(alls):
        table[i + 1, :_pages(n)] = ids[at:at + _pages(n)]
        at += _pages(n)
    q = torch.randn(sum(new), hq, d, generator=g, device=DEV).to(dt)
    s.update(q=q, cache=_cache(g, pages + 2, hkv, d), table=table,
             rows=list(range(1, b + 1)), new=new, alls=alls, out=torch.empty_like(q))
    return s


# ---------------------------------------------------------------- plain forms, 32 bits

def _values(codes, scales):
    """fp32 values of code bytes (..., n/2) and scale bytes (..., n/32)."""
    lut = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0,
                        -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0], device=codes.device)
    x = torch.stack([lut[(codes & 15).int()], lut[(codes >> 4).int()]], dim=-1)
    x = torch.ldexp(x.reshape(*scales.shape, 32), (scales.int() - 127).unsqueeze(-1))
    return x.reshape(*codes.shape[:-1], -1)


def _unpack(blocks, d):
    """fp32 K and V (n, 16, d) of page blocks (n, 17 d)."""
    n, w = blocks.shape[0], min(d, 128)
    kc, vc, ks, vs = blocks.split([8 * d, 8 * d, d // 2, d // 2], dim=1)
    vc = vc.reshape(n, d // w, 4, 16, 4, w // 32).permute(0, 2, 4, 1, 3, 5)
    return (_values(kc.reshape(n, PAGE, d // 2), ks.reshape(n, d // 32, PAGE).transpose(1, 2)),
            _values(vc.reshape(n, PAGE, d // 2), vs.reshape(n, d // 32, PAGE).transpose(1, 2)))


def _gather(cache, pages, d):
    """fp32 K and V (batch, kv_heads, 16 * width, d) of the page ids (batch, width)."""
    b, width = pages.shape
    blocks = cache[pages.long().reshape(-1)]
    out = []
    for x in _unpack(blocks.reshape(-1, 17 * d), d):
        x = x.view(b, width, cache.shape[1], PAGE, d).permute(0, 2, 1, 3, 4)
        out.append(x.reshape(b, cache.shape[1], width * PAGE, d))
    return out


def _attend(q, k, v, seen, cap, sink):
    """fp32 attention of q (batch, kv_heads, rows, d); seen (batch, 1 or rows, keys)."""
    s = torch.matmul(q, k.transpose(2, 3)) * (1.0 / math.sqrt(q.shape[3]))
    if cap:
        s = cap * torch.tanh(s / cap)
    s = s.masked_fill(~seen.unsqueeze(1), float("-inf"))
    top = s.amax(-1, keepdim=True)
    if sink is not None:                                     # (kv_heads, rows)
        top = torch.maximum(top, sink[None, :, :, None])
    p = torch.exp(s - top)
    total = p.sum(-1, keepdim=True)
    if sink is not None:
        total = total + torch.exp(sink[None, :, :, None] - top)
    return torch.matmul(p, v) / total


def _rope(x, positions, inv_freq, style):
    a = positions.double()[:, None] * inv_freq.double()      # far positions: angles in 64 bits
    c, s = a.cos().float()[:, None], a.sin().float()[:, None]
    x = x.float()
    if style == 0:
        x0, x1 = x.chunk(2, dim=-1)
        return torch.cat([x0 * c - x1 * s, x1 * c + x0 * s], dim=-1)
    x0, x1 = x[..., 0::2], x[..., 1::2]
    return torch.stack([x0 * c - x1 * s, x1 * c + x0 * s], dim=-1).flatten(-2)


def _rounded(x):
    """The values that the 4-bit cache holds for x."""
    codes, e = _quantize(x)
    return _values(codes[..., 0::2] | codes[..., 1::2] << 4, e)


def _run_tables(s):
    table, rows, cached, new = s["table"], s["rows"], s["cached"], s["new"]
    b, cap, nt = rows.shape[0], s["capacity"], s["num_tokens"]
    lens = cached + new
    p0, p1 = (cached + PAGE - 1) // PAGE, (lens + PAGE - 1) // PAGE
    taken = torch.cumsum(p1 - p0, 0) - (p1 - p0)
    zero = torch.zeros(1, dtype=torch.int64, device=table.device)
    indptr = torch.cat([zero, torch.cumsum(p1, 0)])
    q_indptr = torch.cat([zero, torch.cumsum(new, 0)])
    each = torch.arange(b, device=table.device)
    req = torch.repeat_interleave(each, p1, output_size=cap)
    j = torch.arange(cap, device=table.device) - indptr[req]
    at = taken[req] + j - p0[req]
    pool = torch.cat([s["new_pages"], s["new_pages"].new_full((1,), -1)])
    fresh = pool[at.clamp(0, pool.shape[0] - 1)]
    ids = torch.where(j >= p0[req], fresh, table[rows[req], j])
    table[rows[req], j] = ids
    treq = torch.repeat_interleave(each, new, output_size=nt)
    pos = cached[treq] + torch.arange(nt, device=table.device) - q_indptr[treq]
    page = table[rows[treq], pos // PAGE]
    slots = torch.where(page >= 0, page * PAGE + pos % PAGE, -1)
    i32 = lambda t: t.to(torch.int32)  # noqa: E731
    return dict(table=table, indptr=i32(indptr), indices=ids,
                last=i32(torch.where(lens > 0, lens - PAGE * (p1 - 1), lens)),
                q_indptr=i32(q_indptr), slots=i32(slots), positions=i32(pos))


def _run_write(s):
    there = (s["slots"] >= 0)[:, None, None]
    q, k, v = s["q"], s["k"], s["v"]
    k4 = _rounded(_rope(k, s["positions"], s["inv_freq"], s["style"]))
    v4 = _rounded(v.float())
    q.copy_(_rope(q, s["positions"], s["inv_freq"], s["style"]))
    return dict(q=q, k=torch.where(there, k4, 0.0).to(k.dtype),
                v=torch.where(there, v4, 0.0).to(v.dtype))


def _run_decode(s):
    q, indptr, d = s["q"], s["indptr"].long(), s["d"]
    b, hkv = q.shape[0], s["hkv"]
    col = torch.arange(s["hint"], device=q.device)
    at = (indptr[:-1, None] + col).clamp(max=s["indices"].shape[0] - 1)
    k, v = _gather(s["cache"], s["indices"][at], d)
    lens = (indptr[1:] - indptr[:-1] - 1) * PAGE + s["last"]
    t = torch.arange(k.shape[2], device=q.device)
    seen = t < lens[:, None]
    if s["window"]:
        seen = seen & (t >= lens[:, None] - s["window"])
    sink = None if s["sink"] is None else s["sink"].view(hkv, -1)
    o = _attend(q.float().view(b, hkv, -1, d), k, v, seen[:, None], s["cap"], sink)
    return o.reshape(q.shape).to(q.dtype)


def _run_extend(s):
    q, d, hkv = s["q"], s["d"], s["hkv"]
    new = torch.tensor(s["new"], device=q.device)
    alls = torch.tensor(s["alls"], device=q.device)
    first = torch.cumsum(new, 0) - new
    i = torch.arange(max(s["new"]), device=q.device)
    at = (first[:, None] + i).clamp(max=q.shape[0] - 1)
    pages = s["table"][torch.tensor(s["rows"], device=q.device)].clamp(min=0)
    k, v = _gather(s["cache"], pages, d)
    pos = (alls - new)[:, None] + i                          # (batch, new)
    t = torch.arange(k.shape[2], device=q.device)
    seen = t <= pos[:, :, None]
    if s["window"]:
        seen = seen & (t > pos[:, :, None] - s["window"])
    b, n, g = pos.shape[0], pos.shape[1], q.shape[1] // hkv
    qq = q.float()[at].view(b, n, hkv, g, d).permute(0, 2, 1, 3, 4).reshape(b, hkv, n * g, d)
    o = _attend(qq, k, v, seen.repeat_interleave(g, dim=1), s["cap"], None)
    o = o.view(b, hkv, n, g, d).permute(0, 2, 1, 3, 4).reshape(b, n, hkv * g, d)
    return o[i < new[:, None]].to(q.dtype)


# ---------------------------------------------------------------- one pass

def run(s):
    op = s["op"]
    if not own:
        return {"tables": _run_tables, "write": _run_write, "decode": _run_decode,
                "extend": _run_extend}[op](s)
    import sys
    if "decode-kernel_amd" not in sys.path:
        sys.path.insert(0, "decode-kernel_amd")
    if op == "tables":
        import paging
        t = paging.grow_block_tables(s["table"], s["rows"], s["cached"], s["new"], s["new_pages"],
                                     s["num_tokens"], s["capacity"])
        return dict(table=s["table"], indptr=t.kv_indptr, indices=t.kv_indices,
                    last=t.kv_last_page_len, q_indptr=t.q_indptr, slots=t.slots,
                    positions=t.positions)
    if op == "write":
        import paging
        paging.write_kv4(s["k"], s["v"], s["cache"], s["slots"], q=s["q"], inv_freq=s["inv_freq"],
                         positions=s["positions"], rope_style=s["style"])
        k, v = paging.read_kv4(s["cache"], s["slots"], s["q"].dtype)
        return dict(q=s["q"], k=k, v=v)
    if op == "decode":
        import attention
        return attention.decode_attention(
            s["q"], s["cache"], s["indptr"], s["indices"], s["last"], split_kv=0,
            max_pages_per_seq=s["hint"], logit_cap=s["cap"], window=s["window"], sinks=s["sink"])
    import extend
    return extend.extend_attention_kv4(s["q"], s["cache"], s["table"], s["rows"], s["new"],
                                       s["alls"], out=s["out"], logit_cap=s["cap"],
                                       window=s["window"])


def work(case):
    op = case["op"]
    if op == "tables":
        b = case["batch"]
        cached, new = zip(*_table_pairs(case))
        live = sum(_pages(c) for c in cached)
        pages = sum(_pages(c + n) for c, n in zip(cached, new))
        # lengths and rows; live entries, new ids; table entries, indices, slots, positions
        return dict(bytes=b * 36 + 4 * (live + 3 * (pages - live) + pages + 2 * sum(new)), flops=0)
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    if op == "write":
        t = case["tokens"] + case["pad"]
        # k and v, q in and out, the cache's bytes, the values that come back
        return dict(bytes=t * d * (4 * hkv + 4 * hq + 17 * hkv / 16 + 4 * hkv) + 8 * t,
                    flops=t * d * (6 * (hq + hkv) / 2 + 8 * hkv))
    if op == "decode":
        lens = _spread(case["lo"], case["hi"], case["batch"])
        if case["window"]:
            lens = [min(n, case["window"]) for n in lens]
        return dict(bytes=sum(_pages(n) for n in lens) * (hkv * 17 * d + 4) +
                    4 * case["batch"] * hq * d, flops=4 * hq * d * sum(lens))
    pre, new = zip(*_pairs(case["prefix_lo"], case["prefix_hi"], case["new_lo"], case["new_hi"],
                           case["batch"]))
    far = case["window"] or 1 << 40
    seen = sum(min(far, p + i + 1) for n, p in zip(new, pre) for i in range(n))
    return dict(bytes=sum(_pages(min(far + n, n + p)) for n, p in zip(new, pre)) * hkv * 17 * d +
                4 * sum(new) * hq * d, flops=4 * hq * d * seen)


# ---------------------------------------------------------------- 64 bits, from the format

def _exact_rows(cache, pages, d, first):
    """fp64 rows (kv_heads, 16 * pages, d): K (first = 0) or V (first = 1) of the page ids."""
    blocks = cache[pages.long()]
    t = torch.arange(PAGE, device=cache.device)[:, None]
    j = torch.arange(d, device=cache.device)[None, :]
    w = min(d, 128)
    if first == 0:
        byte, odd = t * (d // 2) + j // 2, j % 2 == 1
    else:
        c, e = j % w // (w // 16), j % (w // 16)
        byte = 8 * d + j // w * 8 * w + t // 4 * 2 * w + c * (w // 8) + t % 4 * (w // 32) + e // 2
        odd = e % 2 == 1
    code = blocks[:, :, byte].to(torch.int64)
    code = torch.where(odd, code // 16, code % 16)
    scale = blocks[:, :, 16 * d + first * (d // 2) + j // 32 * 16 + t].to(torch.float64)
    size = code % 8                               # 1 sign, 2 exponent, 1 mantissa bits, bias 1
    ex, man = size // 2, (size % 2).double()
    x = torch.where(ex == 0, man / 2, (1 + man / 2) * torch.exp2((ex - 1).double()))
    x = torch.where(code >= 8, -x, x) * torch.exp2(scale - 127)
    return x.transpose(0, 1).reshape(cache.shape[1], -1, d)


def _exact_attend(q, k, v, seen, cap, sink):
    """fp64: q (heads, rows, d), k and v (kv_heads, keys, d), seen (rows, keys)."""
    g = q.shape[0] // k.shape[0]
    out = torch.empty_like(q)
    for h in range(q.shape[0]):
        s = (q[h] @ k[h // g].t()) / math.sqrt(q.shape[2])
        if cap:
            s = torch.tanh(s / cap) * cap
        s = torch.where(seen, s, torch.full_like(s, -math.inf))
        if sink is not None:
            s = torch.cat([s, sink[h].expand(s.shape[0], 1)], dim=1)
        p = torch.softmax(s, dim=1)[:, :k.shape[1]]
        out[h] = p @ v[h // g]
    return out


def _exact_held(x):
    """fp64 values that the cache holds for x: the nearest E2M1 multiple, ties to even."""
    b = x.reshape(*x.shape[:-1], -1, 32)
    man, ex = torch.frexp(b.abs().amax(-1, keepdim=True))   # man in [1/2, 1)
    e = (ex - 1 + (man >= 0.875).to(ex.dtype) - 2).double()
    y = b * torch.exp2(-e)
    step = torch.where(y.abs() < 2, 0.5, torch.where(y.abs() < 4, 1.0, 2.0))
    y = (torch.round(y / step) * step).clamp(-6, 6)
    return (y * torch.exp2(e)).reshape(x.shape)


def exact(case, seed):
    if case["op"] == "tables":
        return None                               # whole numbers
    s = prepare(case, seed)
    d = case["d"]
    if case["op"] == "write":
        ang = s["positions"].double()[:, None, None] * s["inv_freq"].double()

        def turn(x):
            x = x.double()
            even, odd = (x[..., :d // 2], x[..., d // 2:]) if case["style"] == 0 else \
                (x[..., 0::2], x[..., 1::2])
            z = torch.complex(even, odd) * torch.polar(torch.ones_like(ang), ang)
            if case["style"] == 0:
                return torch.cat([z.real, z.imag], dim=-1)
            return torch.view_as_real(z).reshape(x.shape)

        there = (s["slots"] >= 0).double()[:, None, None]
        return dict(q=turn(s["q"]), k=_exact_held(turn(s["k"])) * there,
                    v=_exact_held(s["v"].double()) * there)
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    if case["op"] == "decode":
        sink = None if s["sink"] is None else s["sink"].double()
        ip, last = s["indptr"].tolist(), s["last"].tolist()
        for b in range(case["batch"]):
            pages = s["indices"][ip[b]:ip[b + 1]]
            n = PAGE * (len(pages) - 1) + last[b]
            lo = max(0, n - case["window"]) if case["window"] else 0
            k, v = (_exact_rows(s["cache"], pages, d, f)[:, lo:n] for f in (0, 1))
            seen = torch.ones(1, n - lo, dtype=torch.bool, device=DEV)
            out[b] = _exact_attend(s["q"][b].double()[:, None], k, v, seen, case["cap"], sink)[:, 0]
        return out
    at = 0
    for row, new, n in zip(s["rows"], s["new"], s["alls"]):
        pages = s["table"][row, :_pages(n)]
        k, v = (_exact_rows(s["cache"], pages, d, f)[:, :n] for f in (0, 1))
        pos = torch.arange(n - new, n, device=DEV)[:, None]
        t = torch.arange(n, device=DEV)
        seen = t <= pos
        if case["window"]:
            seen = seen & (t > pos - case["window"])
        q = s["q"][at:at + new].double().transpose(0, 1).contiguous()
        out[at:at + new] = _exact_attend(q, k, v, seen, case["cap"], None).transpose(0, 1)
        at += new
    return out
