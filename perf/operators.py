"""Cases of the 4-bit key/value cache: planning its pages, writing and reading its rows, attention over it.

A cache is a tensor of pages. A page holds `page` tokens of every head; a head's part of it is

    K codes [page][D/2] | V codes [page/4][16][4][D/32 bytes] | K scales [page][D/32] | V scales [page/4][D/32][4]

with D = head_dim padded to 64, 128 or 256. Codes are E2M1 (low nibble = even element), scales one exponent byte for each
32 elements of a token's row. The V codes of four tokens lie together in 16 pieces of D/16 elements, their scales block by
block, so that one load of the attention's value product takes four tokens of its columns.

`own` is set from outside: False computes every operator with elementary torch operations, True calls the framework."""
import math

import torch

own = False

_GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
_MANY = 0.6180339887498949  # ragged lengths: multiples of the golden ratio, taken modulo 1


# ---- sizes ------------------------------------------------------------------------------------------------------

def _width(d):
    return 64 if d <= 64 else 128 if d <= 128 else 256


def _head_bytes(case):
    w = _width(case["head_dim"])
    return case["page"] * (w + w // 16)


def _ragged(n, low, high, turn=0.0):
    """n whole numbers spread over [low, high]; the first is `high`, so that the bound a caller states is met."""
    return [high - int((high - low + 1) * (((i * _MANY) + (turn if i else 0.0)) % 1.0)) if high > low else high for i in range(n)]


def _lengths(case):
    """(cached, new) tokens of each request."""
    n = case["requests"]
    cached = _ragged(n, case["cached_low"], case["cached"])
    new = _ragged(n, case["new_low"], case["new"], 0.37)
    return cached, new


def _ceil(a, b):
    return -(-a // b)


# ---- cases ------------------------------------------------------------------------------------------------------

def listed():
    return [
        # one decode step of a full serving batch: each request gets one token, one in sixteen of them a page
        dict(name="plan_step", op="plan", requests=64, cached_low=1, cached=8192, new_low=1, new=1, page=16),
        # admission of many prompts at once
        dict(name="plan_prompts", op="plan", requests=2048, cached_low=0, cached=100, new_low=1, new=1023, page=64),
        # one token of each request written (and read back)
        dict(name="append_step", op="append", tokens=64, kv_heads=8, head_dim=128, page=16, type="bf16"),
        # a prefill's keys and values, fp32 rows of a width that is padded
        dict(name="append_prompts", op="append", tokens=32771, kv_heads=8, head_dim=96, page=64, type="fp32"),
        # a shared prefix read back to be handed on
        dict(name="read_prefix", op="read", tokens=65537, kv_heads=8, head_dim=128, page=64, type="bf16"),
        # one user, short context: latency
        dict(name="attend_one", op="attend", requests=1, cached_low=1023, cached=1023, new_low=1, new=1, kv_heads=8, group=4, head_dim=128,
             page=16, type="bf16", causal=True),
        # a decode step of a ragged batch: what serving spends its time on
        dict(name="attend_batch", op="attend", requests=48, cached_low=16, cached=8191, new_low=1, new=1, kv_heads=8, group=4, head_dim=128,
             page=64, type="bf16", causal=True),
        # a few long contexts, fp32 queries, an odd group of heads
        dict(name="attend_long_f32", op="attend", requests=3, cached_low=50001, cached=131071, new_low=1, new=1, kv_heads=4, group=7,
             head_dim=64, page=128, type="fp32", causal=True),
        # prompts over what is cached already, causal
        dict(name="attend_prompts", op="attend", requests=4, cached_low=0, cached=2047, new_low=1500, new=2048, kv_heads=8, group=4,
             head_dim=128, page=64, type="bf16", causal=True),
        # a shared memory that short queries read whole: no mask, wide heads
        dict(name="attend_memory", op="attend", requests=16, cached_low=1000, cached=4100, new_low=5, new=33, kv_heads=2, group=8,
             head_dim=256, page=32, type="bf16", causal=False),
        # one query's retrieved rows: latency
        dict(name="selected_one", op="selected", requests=1, cached_low=8000, cached=8000, selected=10, kv_heads=8, group=1, head_dim=128,
             page=64, type="bf16"),
        # a batch of queries, each with the 100 rows that a search over 65,536 of them returned
        dict(name="selected_batch", op="selected", requests=256, cached_low=65536, cached=65536, selected=100, kv_heads=8, group=4,
             head_dim=128, page=64, type="bf16"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("plan", "append", "read", "attend", "attend", "attend", "selected", "selected"))
    page = rng.choice((16, 32, 64, 128))
    if op == "plan":
        n = _log(rng, 1, 2048)
        if rng.random() < 0.5:
            return dict(op=op, requests=n, cached_low=rng.randint(0, 50), cached=_log(rng, 64, 16384), new_low=1, new=1, page=page)
        new = _log(rng, 2, max(2, min(8192, (1 << 20) // n)))
        return dict(op=op, requests=n, cached_low=0, cached=_log(rng, 1, 4096), new_low=rng.randint(0, min(2, new)), new=new, page=page)
    heads, d = rng.choice((1, 2, 3, 4, 8)), rng.choice((64, 64, 80, 96, 112, 128, 128, 192, 256))
    kind = rng.choice(("bf16", "bf16", "fp32"))
    if op in ("append", "read"):
        most = max(64, (32768 * 8 * 128) // (heads * _width(d)))
        return dict(op=op, tokens=_log(rng, 1, most), kv_heads=heads, head_dim=d, page=page, type=kind)
    group = rng.choice((1, 2, 3, 4, 5, 7, 8, 16))
    if op == "selected":
        return dict(op=op, requests=_log(rng, 1, max(1, 1024 // (heads * group) * 4)), cached_low=1000, cached=_log(rng, 2000, 65536),
                    selected=_log(rng, 1, 240), kv_heads=heads, group=group, head_dim=d, page=page, type=kind)
    low = rng.randint(1, 15)
    if rng.random() < 0.6:  # single tokens
        n = _log(rng, 1, 64)
        room = (48 * 4096 * 8 * 128) // (n * heads * _width(d))  # no more cache than the largest listed case reads
        top = _log(rng, 32, max(64, min(131072, room)))
        return dict(op=op, requests=n, cached_low=low, cached=top, new_low=1, new=1, kv_heads=heads, group=group, head_dim=d, page=page,
                    type=kind, causal=True)
    n, top = _log(rng, 1, 16), _log(rng, 16, 4096)
    work = 6e10 / (3 if kind == "fp32" else 1)  # and no more products
    new = max(2, min(2048, int(work / (n * heads * group * _width(d) * (top + 1000)))))
    new = _log(rng, 2, max(2, new))
    return dict(op=op, requests=n, cached_low=0, cached=top, new_low=rng.randint(0, 2), new=new, kv_heads=heads, group=group, head_dim=d,
                page=page, type=kind, causal=rng.random() < 0.75)


# ---- the 4-bit rows, in elementary operations -------------------------------------------------------------------

def _encode(x):
    """(codes, scale bytes) of rows [..., D]: D/2 bytes and D/32 bytes."""
    b = x.float().unflatten(-1, (-1, 32))
    bits = b.abs().amax(-1).view(torch.int32)
    e = ((bits + 0x200000) >> 23) - 2
    e = torch.where(bits >= 0x7F800000, 255, e.clamp(2, 252))
    y = torch.ldexp(b.double(), (127 - e).double()[..., None]).float().nan_to_num(0.0, 0.0, 0.0)  # a power of two: exact
    y = torch.where(e[..., None] == 255, 0.0, y)
    a = y.abs()
    code = (a > 0.25).int() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)
    code = (code + 8 * (y < 0)).flatten(-2).to(torch.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4), e.to(torch.uint8)


def _decode(codes, scales):
    """Rows [..., D] in fp32."""
    grid = torch.tensor(_GRID + tuple(-g for g in _GRID), device=codes.device)
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    s = torch.where(scales == 255, math.nan, torch.exp2(scales.float() - 127.0))
    return (grid[c.int()].unflatten(-1, (-1, 32)) * s[..., None]).flatten(-2)


def _parts(case, heads):
    """Views of a head's bytes [..., head bytes] as (K codes, V codes, K scales, V scales)."""
    p, w = case["page"], _width(case["head_dim"])
    k, v, ks, vs = heads.split((p * w // 2, p * w // 2, p * w // 32, p * w // 32), -1)
    return (k.unflatten(-1, (p, w // 2)), v.unflatten(-1, (p // 4, 16, 4, w // 32)), ks.unflatten(-1, (p, w // 32)), vs.unflatten(-1, (p // 4, w // 32, 4)))


def _write_slots(case, cache, k, v, slots):
    """Rows k, v [tokens, heads, D] into their slots."""
    p = case["page"]
    kc, vc, ks, vs = _parts(case, cache)
    page, at = slots // p, slots % p
    codes, scales = _encode(k)
    kc[page, :, at] = codes
    ks[page, :, at] = scales
    codes, scales = _encode(v)
    vc[page, :, at // 4, :, at % 4] = codes.unflatten(-1, (16, -1))
    vs[page, :, at // 4, :, at % 4] = scales


def _read_slots(case, cache, slots):
    """(keys, values) [..., D] of slots [...], all heads of each."""
    p = case["page"]
    kc, vc, ks, vs = _parts(case, cache)
    page, at = slots // p, slots % p
    return (_decode(kc[page, :, at], ks[page, :, at]), _decode(vc[page, :, at // 4, :, at % 4].flatten(-2), vs[page, :, at // 4, :, at % 4]))


def _read_pages(case, cache, tables):
    """(keys, values) [requests, heads, tokens, D] of whole block tables [requests, pages]."""
    kc, vc, ks, vs = _parts(case, cache[tables])
    k = _decode(kc, ks)                                                   # [requests, pages, heads, page, D]
    v = _decode(vc.transpose(-2, -3).flatten(-2).flatten(-3, -2), vs.transpose(-1, -2).flatten(-3, -2))
    return k.transpose(1, 2).flatten(2, 3), v.transpose(1, 2).flatten(2, 3)


def _softmax_sum(s, seen, v):
    """(sum of softmax(s) v, log of the sum of exponentials) over the last axis of s, where `seen`; 0 and -inf where nothing is."""
    s = torch.where(seen, s, -math.inf)
    top = s.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = torch.exp(s - top)
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v) / torch.where(total > 0, total, 1.0)
    return out, (top + torch.log(total))[..., 0]


# ---- inputs -----------------------------------------------------------------------------------------------------

_TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def _ints(values, kind=torch.int32):
    return torch.tensor(values, dtype=kind, device="cuda")


def _normal(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda")


def _rows(case, gen, n):
    """n rows of every head, padded with zeros: normal, a few channels larger than the others, as keys are."""
    d, w = case["head_dim"], _width(case["head_dim"])
    x = _normal(gen, n, case["kv_heads"], d)
    x[..., 3::41] *= 5.0
    return torch.nn.functional.pad(x, (0, w - d))


def _filled(case, gen, pages):
    """A cache of `pages` pages, every token of them written (the ones behind a request's last are what was there before)."""
    cache = torch.empty((pages, case["kv_heads"], _head_bytes(case)), dtype=torch.uint8, device="cuda")
    p, part = case["page"], max(1, (1 << 17) // (case["page"] * case["kv_heads"]))
    for at in range(0, pages, part):
        m = min(part, pages - at)
        slots = torch.arange(m * p, device="cuda")
        _write_slots(case, cache[at:at + m], _rows(case, gen, m * p), _rows(case, gen, m * p), slots)
    return cache


def _tables(case, gen, lengths):
    """Block tables of requests with these lengths over shuffled pages, and the number of pages."""
    p = case["page"]
    stride = max(1, max(_ceil(x, p) for x in lengths))
    pages = sum(_ceil(x, p) for x in lengths) + 3
    order = torch.randperm(pages, generator=gen, device="cuda")
    need = _ints([_ceil(x, p) for x in lengths], torch.int64)
    first = torch.cumsum(need, 0) - need
    at = torch.arange(stride, device="cuda")
    take = torch.where(at < need[:, None], first[:, None] + at, 0)
    return torch.where(at < need[:, None], order[take], pages - 1).to(torch.int32), pages


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    s = dict(case=dict(case))
    if case["op"] == "plan":
        p = case["page"]
        cached, new = _lengths(case)
        total = sum(new)
        need = [_ceil(c + a, p) - _ceil(c, p) for c, a in zip(cached, new)]
        held = sum(_ceil(c, p) for c in cached)
        ring = held + sum(need) + 17
        order = torch.randperm(ring, generator=gen, device="cuda").to(torch.int32)
        stride = max(1, max(_ceil(c + a, p) for c, a in zip(cached, new)))
        s.update(lengths=_ints(cached), new=_ints(new), ring=order, cursor=_ints([held, ring], torch.int64), pages=ring,
                 slot_cap=total + total // 8 + 1)
        have = _ints([_ceil(c, p) for c in cached], torch.int64)
        first = torch.cumsum(have, 0) - have
        at = torch.arange(stride, device="cuda")
        take = torch.where(at < have[:, None], first[:, None] + at, 0)
        s["tables"] = torch.where(at < have[:, None], order[take], -1).to(torch.int32)
        s["out"] = dict(starts=torch.empty(len(new) + 1, dtype=torch.int32, device="cuda"),
                        slots=torch.empty(s["slot_cap"], dtype=torch.int64, device="cuda"), lengths=torch.empty_like(s["lengths"]),
                        cursor=torch.empty_like(s["cursor"]), status=torch.empty(4, dtype=torch.int32, device="cuda"), tables=s["tables"])
        return s
    kind, d = _TYPES[case["type"]], case["head_dim"]
    if case["op"] in ("append", "read"):
        t, pages = case["tokens"], _ceil(case["tokens"], case["page"]) + 2
        order = torch.randperm(pages, generator=gen, device="cuda")  # a prompt's tokens lie together, page after page
        at = torch.arange(t, device="cuda")
        s["slots"] = order[at // case["page"]] * case["page"] + at % case["page"]
        if case["op"] == "append":
            s["cache"] = torch.zeros((pages, case["kv_heads"], _head_bytes(case)), dtype=torch.uint8, device="cuda")
            s["k"], s["v"] = (_rows(case, gen, t)[..., :d].to(kind).contiguous() for _ in range(2))
        else:
            s["cache"] = _filled(case, gen, pages)
        s["out"] = [torch.empty((t, case["kv_heads"], d), dtype=kind, device="cuda") for _ in range(2)]
        return s
    heads = case["kv_heads"] * case["group"]
    if case["op"] == "attend":
        cached, new = _lengths(case)
        lengths = [c + a for c, a in zip(cached, new)]
        starts = [sum(new[:i]) for i in range(len(new) + 1)]
        s.update(starts=_ints(starts), rows=starts[-1], max_new=max(new))
    else:
        n = case["requests"]
        lengths = [case["cached"]] * n  # one memory that every request reads
        s.update(rows=n)
    s.update(lengths=_ints(lengths), max_length=max(lengths))
    if case["op"] == "attend":
        s["tables"], pages = _tables(case, gen, lengths)
    else:
        table, pages = _tables(case, gen, lengths[:1])
        s["tables"] = table.expand(len(lengths), -1).contiguous()
        n, k = case["requests"], case["selected"]
        # distinct rows in no order; every seventh list is shorter, as a search that finds fewer returns it
        part = case["cached"] // k
        some = torch.randint(0, part, (case["kv_heads"], n, k), generator=gen, device="cuda")
        ids = some * k + torch.arange(k, device="cuda").flip(0)
        counts = torch.full((case["kv_heads"], n), k, dtype=torch.int32, device="cuda")
        counts.view(-1)[6::7] = k // 2
        s["ids"] = torch.where(torch.arange(k, device="cuda") < counts[..., None], ids, -1)
        s["counts"] = counts
    s["cache"] = _filled(case, gen, pages)
    # keys meet queries that single some of them out: scores of a standard deviation of about 3
    s["q"] = (2.0 * _normal(gen, s["rows"], heads, d)).to(kind)
    s["out"] = dict(out=torch.empty((s["rows"], heads, d), dtype=kind, device="cuda"),
                    lse=torch.empty((s["rows"], heads), dtype=torch.float32, device="cuda"))
    return s


# ---- the plain forms --------------------------------------------------------------------------------------------

def _plan_plain(s):
    case, p = s["case"], s["case"]["page"]
    cached, new = s["lengths"].long(), s["new"].long()
    have, want = (cached + p - 1) // p, (cached + new + p - 1) // p
    need = want - have
    before = torch.cumsum(need, 0) - need
    ends = torch.cumsum(new, 0)
    starts = torch.cat((ends.new_zeros(1), ends))
    ring = s["ring"].numel()
    stride = s["tables"].shape[1]
    at = torch.arange(stride, device="cuda")
    fresh = (at >= have[:, None]) & (at < want[:, None])
    take = (s["cursor"][0] + before[:, None] + at - have[:, None]) % ring
    tables = torch.where(fresh, s["ring"][take], s["tables"])
    t = torch.arange(s["slot_cap"], device="cuda")
    req = torch.searchsorted(ends, t, right=True)
    live = req < new.numel()
    req = torch.where(live, req, 0)
    pos = cached[req] + t - starts[req]
    page = tables[req, torch.where(live, pos // p, 0)].long()
    slots = torch.where(live, page * p + pos % p, -1)
    taken = need.sum()
    return dict(starts=starts.int(), slots=slots, lengths=(cached + new).int(), cursor=torch.stack((s["cursor"][0] + taken, s["cursor"][1])),
                status=torch.stack((taken * 0, taken, ends[-1], taken * 0)).int(), tables=tables)


def _attend_plain(s):
    case = s["case"]
    h, g, d, w = case["kv_heads"], case["group"], case["head_dim"], _width(case["head_dim"])
    n, m = case["requests"], s["max_new"]
    starts, lengths = s["starts"].long(), s["lengths"].long()
    new = starts[1:] - starts[:-1]
    j = torch.arange(m, device="cuda")
    row = torch.where(j < new[:, None], starts[:-1, None] + j, 0)
    q = torch.nn.functional.pad(s["q"].float(), (0, w - d))[row]                                   # [n, m, heads, D]
    q = q.unflatten(2, (h, g)).permute(0, 2, 1, 3, 4).flatten(2, 3) / math.sqrt(d)                 # [n, h, m g, D]
    k, v = _read_pages(case, s["cache"], s["tables"].long())
    score = torch.matmul(q, k.transpose(-1, -2).contiguous())
    del k
    limit = (lengths - new + 1)[:, None] + j if case["causal"] else lengths[:, None].expand(-1, m)
    seen = torch.arange(v.shape[2], device="cuda") < limit.repeat_interleave(g, 1)[:, None, :, None]
    out, lse = _softmax_sum(score, seen, v)
    out, lse = out.unflatten(2, (m, g)).transpose(1, 2).flatten(2, 3), lse.unflatten(2, (m, g)).transpose(1, 2).flatten(2, 3)
    live = j < new[:, None]
    return dict(out=out[live][..., :d].to(s["q"].dtype), lse=lse[live])


def _selected_plain(s):
    case = s["case"]
    h, g, d, w, p = case["kv_heads"], case["group"], case["head_dim"], _width(case["head_dim"]), case["page"]
    n, k = case["requests"], case["selected"]
    seen = (torch.arange(k, device="cuda") < s["counts"][..., None]) & (s["ids"] >= 0) & (s["ids"] < s["lengths"][None, :, None])
    ids = torch.where(seen, s["ids"], 0)
    page = torch.gather(s["tables"].long()[None].expand(h, -1, -1), 2, ids // p)
    at = ids % p
    kc, vc, ks, vs = _parts(case, s["cache"])
    head = torch.arange(h, device="cuda")[:, None, None]
    key = _decode(kc[page, head, at], ks[page, head, at])                                          # [h, n, k, D]
    val = _decode(vc[page, head, at // 4, :, at % 4].flatten(-2), vs[page, head, at // 4, :, at % 4])
    q = torch.nn.functional.pad(s["q"].float(), (0, w - d)).unflatten(1, (h, g)).transpose(0, 1) / math.sqrt(d)
    score = torch.matmul(q, key.transpose(-1, -2).contiguous())                                    # [h, n, g, k]
    out, lse = _softmax_sum(score, seen[:, :, None], val)
    return dict(out=out.transpose(0, 1).flatten(1, 2)[..., :d].to(s["q"].dtype), lse=lse.transpose(0, 1).flatten(1, 2))


def _plain(s):
    op, d = s["case"]["op"], s["case"]["head_dim"] if "head_dim" in s["case"] else 0
    if op == "plan":
        return _plan_plain(s)
    if op == "append":
        pad = _width(d) - d
        k, v = (torch.nn.functional.pad(s[x].float(), (0, pad)) for x in "kv")
        _write_slots(s["case"], s["cache"], k, v, s["slots"])
    if op in ("append", "read"):
        return [x[..., :d].to(s["out"][0].dtype) for x in _read_slots(s["case"], s["cache"], s["slots"])]
    return _attend_plain(s) if op == "attend" else _selected_plain(s)


# ---- the framework's calls --------------------------------------------------------------------------------------

def _own(s):
    import zvdb_amd as zv
    case, out, at = s["case"], s["out"], torch.cuda.current_stream().cuda_stream
    if "layout" not in s:
        pages = s["pages"] if case["op"] == "plan" else s["cache"].shape[0]
        s["layout"] = zv.KVLayout(head_dim=case.get("head_dim", 64), kv_heads=case.get("kv_heads", 1), page_size=case["page"], pages=pages)
        s["type"] = zv.KV_F32 if case.get("type") == "fp32" else zv.KV_BF16
    lay, kind = s["layout"], s["type"]
    if case["op"] == "plan":
        lay.plan_dev(s["lengths"].data_ptr(), s["new"].data_ptr(), case["requests"], s["ring"].data_ptr(), s["ring"].numel(),
                     s["cursor"].data_ptr(), s["tables"].data_ptr(), s["tables"].shape[1], out["starts"].data_ptr(), out["slots"].data_ptr(),
                     s["slot_cap"], out["lengths"].data_ptr(), out["cursor"].data_ptr(), out["status"].data_ptr(), at)
        return out
    if case["op"] in ("append", "read"):
        t, step = case["tokens"], case["kv_heads"] * case["head_dim"]
        if case["op"] == "append":
            lay.append_dev(s["cache"].data_ptr(), s["k"].data_ptr(), step, s["v"].data_ptr(), step, kind, t, s["slots"].data_ptr(), at)
        lay.read_dev(s["cache"].data_ptr(), s["slots"].data_ptr(), t, out[0].data_ptr(), out[1].data_ptr(), kind, at)
        return out
    heads, scale = case["kv_heads"] * case["group"], 1.0 / math.sqrt(case["head_dim"])
    if case["op"] == "attend":
        if "space" not in s:
            s["space"] = torch.empty(lay.attend_workspace(kind, heads, case["requests"], s["rows"], s["max_new"], s["max_length"]),
                                     dtype=torch.uint8, device="cuda")
        lay.attend_dev(s["cache"].data_ptr(), s["q"].data_ptr(), heads * case["head_dim"], kind, heads, case["requests"], s["starts"].data_ptr(),
                       s["rows"], s["max_new"], s["lengths"].data_ptr(), s["tables"].data_ptr(), s["tables"].shape[1], s["max_length"], scale,
                       case["causal"], s["space"].data_ptr(), s["space"].numel(), out["out"].data_ptr(), out["lse"].data_ptr(), at)
        return out
    lay.attend_selected_dev(s["cache"].data_ptr(), s["q"].data_ptr(), heads * case["head_dim"], kind, heads, case["requests"],
                            s["ids"].data_ptr(), s["counts"].data_ptr(), case["selected"], s["lengths"].data_ptr(), s["tables"].data_ptr(),
                            s["tables"].shape[1], scale, out["out"].data_ptr(), out["lse"].data_ptr(), at)
    return out


def run(s):
    return _own(s) if own else _plain(s)


# ---- what a pass cannot do without ------------------------------------------------------------------------------

def work(case):
    if case["op"] == "plan":
        cached, new = _lengths(case)
        pages = sum(_ceil(c + a, case["page"]) - _ceil(c, case["page"]) for c, a in zip(cached, new))
        total, n = sum(new), case["requests"]
        return dict(bytes=8 * n + 8 * pages + 8 * (total + total // 8 + 1) + 8 * n + 40, flops=0)
    d, w, h = case["head_dim"], _width(case["head_dim"]), case["kv_heads"]
    size = 4 if case["type"] == "fp32" else 2
    row = w + w // 16  # a token's key and value of one head
    if case["op"] in ("append", "read"):
        t = case["tokens"]
        values = 2 * t * h * d * size
        return dict(bytes=8 * t + (2 * values + 2 * t * h * row if case["op"] == "append" else values + t * h * row), flops=0)
    g = case["group"]
    if case["op"] == "attend":
        cached, new = _lengths(case)
        rows, tokens, pairs, pages = sum(new), 0, 0, 0
        for c, a in zip(cached, new):
            if a:
                tokens += c + a
                pages += _ceil(c + a, case["page"])
                pairs += a * c + a * (a + 1) // 2 if case["causal"] else a * (c + a)
        bound = h * tokens * row + 4 * pages
    else:
        rows, n, k = case["requests"], case["requests"], case["selected"]
        short = len(range(6, h * n, 7))
        pairs = (h * n * k - short * (k - k // 2)) / h
        bound = h * pairs * row + 8 * h * n * k + 4 * h * n
    return dict(bytes=bound + rows * h * g * (2 * d * size + 4) + 8 * case["requests"], flops=4.0 * d * h * g * pairs)


# ---- the definition in 64 bits ----------------------------------------------------------------------------------

def _value64(code, scale):
    """The number that an E2M1 code and its exponent byte stand for, from its bits."""
    mant, ex = (code & 1).double(), ((code >> 1) & 3).double()
    mag = torch.where(ex == 0, 0.5 * mant, (1.0 + 0.5 * mant) * torch.exp2(ex - 1.0))
    val = torch.where((code & 8) != 0, -mag, mag) * torch.exp2(scale.double() - 127.0)
    return torch.where(scale == 255, math.nan, val)


def _head64(case, cache, h, pages, at):
    """Keys and values in 64 bits of one head's tokens: token i lies in page pages[i], at place at[i]; from the format's offsets."""
    p, d, w = case["page"], case["head_dim"], _width(case["head_dim"])
    e = torch.arange(d, device="cuda")
    flat = cache.reshape(-1)
    base = ((pages * case["kv_heads"] + h) * _head_bytes(case))[:, None]
    t, half, piece = at[:, None], p * w // 2, w // 16
    key_at = base + t * (w // 2) + e // 2
    val_at = base + half + (t // 4) * (2 * w) + (e // piece) * (piece * 2) + (t % 4) * (piece // 2) + (e % piece) // 2
    key_s = base + 2 * half + t * (w // 32) + e // 32
    val_s = base + 2 * half + p * (w // 32) + (t // 4) * (w // 8) + (e // 32) * 4 + t % 4
    shift = (4 * (e % 2)).to(torch.uint8)
    return (_value64((flat[key_at] >> shift) & 15, flat[key_s]), _value64((flat[val_at] >> shift) & 15, flat[val_s]))


def _one64(q, key, val, seen):
    """Attention of rows q [r, d] over key, val [t, d] where seen [r, t], in 64 bits."""
    s = (q @ key.T.contiguous()) / math.sqrt(q.shape[-1])
    s = s.masked_fill(~seen, -math.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.where(seen, torch.exp(s - torch.where(lse == -math.inf, 0.0, lse)[:, None]), 0.0)
    return p @ val, lse


def exact(case, seed):
    if case["op"] == "plan":
        return None  # whole numbers
    s = prepare(case, seed)
    if case["op"] == "append":
        out = []
        for x in (s["k"], s["v"]):
            b = torch.nn.functional.pad(x.double(), (0, _width(case["head_dim"]) - case["head_dim"])).unflatten(-1, (-1, 32))
            top = b.abs().amax(-1, keepdim=True)
            m, e = torch.frexp(top)                           # top = m 2^e, 1/2 <= m < 1
            e = torch.where(m >= 0.875, e, e - 1).double() - 2  # the power of two under it, doubled from 7/4 of it on, over E2M1's 4
            e = torch.where(top == 0, -125.0, e.clamp(-125, 125))
            grid = torch.tensor(_GRID, dtype=torch.float64, device="cuda")
            y = b.abs() / torch.exp2(e)
            far = (y[..., None] - grid).abs()
            far = far * 2 + torch.arange(8, device="cuda") % 2 * 1e-9  # a tie goes to the even code
            out.append((torch.copysign(grid[far.argmin(-1)], b) * torch.exp2(e)).flatten(-2)[..., :case["head_dim"]])
        return out
    d, p, g = case["head_dim"], case["page"], case["group"] if "group" in case else 1
    if case["op"] == "read":
        pages, at = s["slots"] // p, s["slots"] % p
        both = [_head64(case, s["cache"], h, pages, at) for h in range(case["kv_heads"])]
        return [torch.stack([b[i] for b in both], 1) for i in range(2)]
    out = torch.zeros(s["out"]["out"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(s["out"]["lse"].shape, -math.inf, dtype=torch.float64, device="cuda")
    if case["op"] == "attend":
        cached, new = _lengths(case)
        at = 0
        for i in range(case["requests"]):
            a, length = new[i], cached[i] + new[i]
            t = torch.arange(length, device="cuda")
            j = torch.arange(a, device="cuda").repeat_interleave(g)
            seen = t < (length - a + 1 + j if case["causal"] else torch.full_like(j, length))[:, None]
            for h in range(case["kv_heads"] if a else 0):
                key, val = _head64(case, s["cache"], h, s["tables"][i].long()[t // p], t % p)
                o, l = _one64(s["q"][at:at + a, h * g:(h + 1) * g].reshape(a * g, d).double(), key, val, seen)
                out[at:at + a, h * g:(h + 1) * g], lse[at:at + a, h * g:(h + 1) * g] = o.view(a, g, d), l.view(a, g)
            at += a
        return dict(out=out, lse=lse)
    table = s["tables"][0].long()
    for h in range(case["kv_heads"]):
        flat = s["ids"][h].clamp(min=0).reshape(-1)
        key, val = (x.view(case["requests"], case["selected"], d) for x in _head64(case, s["cache"], h, table[flat // p], flat % p))
        for i in range(case["requests"]):
            c = int(s["counts"][h, i])
            if c:
                o, l = _one64(s["q"][i, h * g:(h + 1) * g].double(), key[i, :c], val[i, :c], torch.ones((g, c), dtype=torch.bool, device="cuda"))
                out[i, h * g:(h + 1) * g], lse[i, h * g:(h + 1) * g] = o, l
    return dict(out=out, lse=lse)
