"""A KV cache held in 4 bits: the operators that write it and attend over it, as measurable cases.

The cache (one layer's pool) is ``uint8 [slots, 2 * Hkv, D / 2 + 2]``: 16 consecutive slots form a block, the codes of
its heads (K heads, then V heads; ``8 * D`` bytes each) followed by a 16-bit word per head and slot. A row's word is the fp16
number of its scale s, whose last four bits are 0, with the zero point z in those bits; a code c stands for s * (c - z).
A row x is quantised over its own range, 0 included:

    lo = min(0, min x), hi = max(0, max x), s = (hi - lo) / 15 rounded up to 7 significant bits,
    z = rint(-lo / s), c = clamp(rint(x / s) + z, 0, 15)                  (halves to even)

so that every value is an fp16 number. Inside a block, a K head holds slot after slot; dword w of a slot its elements 8w .. 8w+7,
element 8w + 2i in nibble i and 8w + 2i + 1 in nibble 4 + i. A V head holds, for four slots at a time and for each of 16
columns of D / 16 elements, the 16-bit units of the four slots (see ``_byte_of``).

* ``append``: the QKV projection's epilogue (per-head RMSNorm, rotary embedding) and the append of K and V to the cache, or the
  append alone; what comes back is q and the pages that were written, as the values they hold.
* ``decode``: one new token per sequence attends over its cached history; with ``append`` the token's K and V are stored on the
  way, and the pages they went to come back too.
* ``prefill``: the rows of prompts or chunks attend causally over their history and themselves.
"""

import math

import torch

own = False

DEVICE = "cuda:0"
BLOCK = 16                       # slots of a block
HEADS = ((64, 8, 128), (16, 8, 128), (32, 4, 128), (32, 8, 64))     # query heads, kv heads, head dim


def _append(name, heads, tokens, norm, rope, page=16, idle=0):
    """``tokens`` rows, the last ``idle`` of which are padding (no slot)."""
    hq, hkv, d = heads
    return {"name": name, "op": "append", "hq": hq, "hkv": hkv, "d": d, "tokens": tokens, "norm": norm, "rope": rope,
            "page": page, "idle": idle}


def _decode(name, heads, batch, lo, hi, append, page=16, idle=0, lengths=1):
    """``batch`` sequences of lo..hi tokens, this step's among them (``lengths`` seeds which); the last ``idle`` are empty rows
    of a padded batch."""
    hq, hkv, d = heads
    return {"name": name, "op": "decode", "hq": hq, "hkv": hkv, "d": d, "batch": batch, "lo": lo, "hi": hi,
            "append": append, "page": page, "idle": idle, "lengths": lengths}


def _prefill(name, heads, batch, lo, hi, history, page=16, lengths=1):
    """``batch`` chunks of lo..hi rows (``lengths`` seeds which); ``history``: the longest cached history, the others are at
    least a quarter of it."""
    hq, hkv, d = heads
    return {"name": name, "op": "prefill", "hq": hq, "hkv": hkv, "d": d, "batch": batch, "lo": lo, "hi": hi,
            "history": history, "page": page, "lengths": lengths}


def listed():
    return [
        # one user's decode step on a small model: nothing but latency
        _append("append-1", HEADS[1], 1, True, True),
        # the serving batch's decode step, four rows of padding among it
        _append("append-32", HEADS[0], 36, True, True, idle=4),
        # a chunk of a model without QK norm, narrow heads, larger pages
        _append("append-chunk-hd64", HEADS[3], 1111, False, True, page=64),
        # eight prompts' worth of tokens
        _append("append-prompts", HEADS[0], 10366, True, True),
        # one user's history
        _decode("decode-1", HEADS[1], 1, 778, 778, True),
        # a handful of users, narrow heads, larger pages, two idle rows
        _decode("decode-12-hd64", HEADS[3], 14, 100, 3000, True, page=64, idle=2, lengths=7),
        # the serving batch: 32 sequences of 256 to 4096 tokens
        _decode("decode-32", HEADS[0], 32, 256, 4096, True),
        # long contexts, many of them
        _decode("decode-64-long", HEADS[2], 64, 4096, 16384, False),
        # one request's short chunk behind a cached history
        _prefill("chunk-64", HEADS[1], 1, 64, 64, 2000),
        # chunked prefill of a long document
        _prefill("chunk-512", HEADS[0], 1, 512, 512, 7601),
        # four requests' chunks together, narrow heads, larger pages
        _prefill("chunks-4-hd64", HEADS[3], 4, 1, 512, 8000, page=64, lengths=19),
        # fresh prompts
        _prefill("prompts-8", HEADS[0], 8, 128, 2048, 0, lengths=3),
    ]


def _between(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("append", "decode", "decode", "prefill"))
    heads = rng.choice(HEADS)
    page = rng.choice((16, 16, 32, 64, 128, 256))
    if op == "append":
        tokens = _between(rng, 1, 10000)
        c = _append("", heads, tokens, rng.random() < 0.5, rng.random() < 0.7, page,
                    rng.choice((0, 0, min(3, tokens - 1))))
    elif op == "decode":
        hi = _between(rng, 1, 16000)
        batch = _between(rng, 1, max(1, min(256, 2400000 // (hi * heads[1]))))
        c = _decode("", heads, batch, max(1, hi // rng.choice((1, 4, 100))), hi, rng.random() < 0.5, page,
                    rng.choice((0, 0, min(2, batch - 1))), rng.randrange(1000))
    else:
        pairs = 350000000 // heads[0]              # of rows and keys, about as many as the longest prompts above have
        history = rng.choice((0, _between(rng, 1, 8000)))
        hi = _between(rng, 1, min(2000, pairs // (history + 1000)))
        batch = _between(rng, 1, max(1, min(16, 8192 // hi, pairs // (hi * (hi // 2 + history + 1)))))
        c = _prefill("", heads, batch, max(1, hi // rng.choice((1, 8))), hi, history, page,
                     rng.randrange(1000))
    del c["name"]
    return c


# ---- the layout ----------------------------------------------------------------------------------------------------------------

def _block_bytes(c):
    return 2 * c["hkv"] * (8 * c["d"] + 2 * BLOCK)


def _held(raw, c):
    """float32 [..., 16, 2 * Hkv, D]: the values of blocks of bytes [..., block bytes]."""
    h, d, lead = c["hkv"], c["d"], raw.shape[:-1]
    codes = raw[..., : 16 * h * d]
    nibbles = torch.stack((codes & 15, codes >> 4), -1)                       # in the order of their bits
    k = nibbles[..., : 8 * h * d, :].reshape(*lead, h, BLOCK, d // 8, 2, 4)   # ..., dword, odd elements, nibble
    k = k.transpose(-1, -2).reshape(*lead, h, BLOCK, d)
    v = nibbles[..., 8 * h * d:, :].reshape(*lead, h, 4, 16, 2, d // 64, 2, 4)  # ..., fours, column, pair, unit, of pair, nibble
    n = len(lead)
    order = [n + i for i in (0, 1, 3, 5, 2, 6, 4)]                            # head, slot (fours, pair, of pair), element
    v = v.permute(*range(n), *order).reshape(*lead, h, BLOCK, d)
    words = raw[..., 16 * h * d:].reshape(*lead, 2 * h, BLOCK, 2).to(torch.int32)
    words = words[..., 0] + 256 * words[..., 1]
    scale = (words & 0xFFF0).to(torch.int16).view(torch.float16).float()
    zero = (words & 15).float()
    both = torch.cat((k, v), -3).float()
    return ((both - zero.unsqueeze(-1)) * scale.unsqueeze(-1)).transpose(-2, -3)


def _places(slots, c):
    """Where the bytes of a slot's rows are in a pool: its codes [T, 2 * Hkv, D / 2], its words [T, 2 * Hkv, 2]."""
    h, d, dev = c["hkv"], c["d"], slots.device
    at = lambda n: torch.arange(n, device=dev)  # noqa: E731
    t = (slots % BLOCK).view(-1, 1, 1)
    base = (slots // BLOCK * _block_bytes(c)).view(-1, 1, 1)
    k = at(h).view(1, -1, 1) * 8 * d + t * (d // 2) + at(d // 2)
    units = d // 64
    column = at(16).view(-1, 1, 1) * (d // 8) + at(units).view(1, -1, 1) * 4 + at(2)
    v = (h + at(h)).view(1, -1, 1) * 8 * d + t // 4 * 2 * d + t // 2 % 2 * (4 * units) + t % 2 * 2 + column.reshape(1, 1, -1)
    words = 16 * h * d + (at(2 * h).view(1, -1, 1) * BLOCK + t) * 2 + at(2)
    return base + torch.cat((k, v), 1), base + words


def _quantised(x):
    """Codes and words (scale and zero point) of rows x [..., D] in float32."""
    x = torch.nan_to_num(x, nan=0.0, posinf=57344.0, neginf=-57344.0).clamp(-57344.0, 57344.0)
    lo, hi = x.amin(-1, keepdim=True).clamp(max=0.0), x.amax(-1, keepdim=True).clamp(min=0.0)
    step = (hi - lo) / torch.full_like(lo, 15.0)
    up = ((step.view(torch.int32) + 0x1FFFF) & ~0x1FFFF).view(torch.float32)
    scale = torch.where(step < 2.0 ** -14, torch.ceil(step * 2.0 ** 20) * 2.0 ** -20, up)
    safe = torch.where(scale > 0, scale, torch.ones_like(scale))
    zero = torch.round(-lo / safe)
    code = (torch.round(x / safe) + zero).clamp(0, 15)
    word = (scale.to(torch.float16).view(torch.int16).to(torch.int32) & 0xFFFF) + zero.to(torch.int32)
    return code.to(torch.uint8), word.squeeze(-1)


def _store(pool, slots, k, v, c):
    """Appends rows k, v [T, Hkv, D] (float32); a slot outside the pool is a row of padding."""
    h, d = c["hkv"], c["d"]
    slots = slots.long()
    there = ((slots >= 0) & (slots < pool.shape[0])).nonzero().squeeze(-1)
    slots = slots[there]
    code, word = _quantised(torch.cat((k, v), 1)[there])
    t = code.shape[0]
    kn = code[:, :h].reshape(t, h, d // 8, 4, 2).transpose(-1, -2).reshape(t, h, d // 2, 2)
    vn = code[:, h:].reshape(t, h, 16, 4, d // 64).transpose(-1, -2).reshape(t, h, d // 2, 2)
    n = torch.cat((kn, vn), 1)
    code_at, word_at = _places(slots, c)
    flat = pool.view(-1)
    flat[code_at] = n[..., 0] | (n[..., 1] << 4)
    flat[word_at] = torch.stack((word & 255, word >> 8), -1).to(torch.uint8)


def _pages(pool, pages, c):
    """float32 [pages * page size, 2 * Hkv, D]: what the pages hold."""
    per = c["page"] // BLOCK
    blocks = pages.long().view(-1, 1) * per + torch.arange(per, device=pages.device)
    return _held(pool.view(-1, _block_bytes(c))[blocks.view(-1)], c).reshape(-1, 2 * c["hkv"], c["d"])


# ---- inputs --------------------------------------------------------------------------------------------------------------------

def _pool(c, pages, g):
    """A pool that has served for a while: rows of normal values, about as wide as normalised K and V are."""
    h, d = c["hkv"], c["d"]
    blocks = pages * c["page"] // BLOCK
    nibbles = (torch.randn(65536, 4, generator=g, device=DEVICE) * 3.3 + 7.5).round().clamp(0, 15).to(torch.int32)
    four = (nibbles[:, 0] | nibbles[:, 1] << 4 | nibbles[:, 2] << 8 | nibbles[:, 3] << 12).to(torch.int16)
    pick = torch.randint(0, 65536, (blocks, 8 * h * d), generator=g, device=DEVICE, dtype=torch.int32)
    codes = four[pick].view(torch.uint8)
    del pick
    scale = 0.34 * torch.exp(0.3 * torch.randn(blocks, 2 * h * BLOCK, generator=g, device=DEVICE))
    word = (scale.half().view(torch.int16) & -16) | torch.randint(6, 10, scale.shape, generator=g, device=DEVICE, dtype=torch.int16)
    return torch.cat((codes, word.view(torch.uint8)), 1).view(pages * c["page"], 2 * h, d // 2 + 2)


def _lengths(lo, hi, n, g):
    """n lengths of lo..hi, the longest exactly hi."""
    x = torch.randint(lo, hi + 1, (n,), generator=g)
    x[int(torch.randint(0, n, (1,), generator=g))] = hi
    return x


def _rows_and_keys(c):
    """Per sequence of a decode or prefill case: query rows, and the keys the last of them sees."""
    g = torch.Generator().manual_seed(c["lengths"])
    if c["op"] == "decode":
        keys = torch.zeros(c["batch"], dtype=torch.int64)
        live = c["batch"] - c["idle"]
        keys[:live] = _lengths(c["lo"], c["hi"], live, g)
        return torch.ones_like(keys), keys
    rows = _lengths(c["lo"], c["hi"], c["batch"], g)
    return rows, rows + _lengths(c["history"] // 4, c["history"], c["batch"], g)


def prepare(case, seed):
    c = dict(case)
    g, host = torch.Generator(DEVICE).manual_seed(seed), torch.Generator().manual_seed(seed)
    hq, h, d, page = c["hq"], c["hkv"], c["d"], c["page"]
    randn = lambda *shape: torch.randn(shape, generator=g, device=DEVICE)  # noqa: E731
    s = {"case": c}
    if c["op"] == "append":
        t, live = c["tokens"], c["tokens"] - c["idle"]
        # prompts and chunks fill pages front to back; a decode step's rows go to pages of their own
        per = page if live > 256 else 1
        used = -(-live // per)
        pages = used + used // 8 + 1
        order = torch.randperm(pages, generator=host)[:used]
        first = 0 if per > 1 else torch.randint(0, page, (used,), generator=host)
        slots = torch.full((t,), -1, dtype=torch.int64)
        i = torch.arange(live)
        slots[:live] = order[i // per] * page + (i % per if per > 1 else first)
        s["pool"] = _pool(c, pages, g)
        s["slots"], s["pages"] = slots.to(DEVICE, torch.int32), order.to(DEVICE, torch.int32)
        s["q"], s["k"], s["v"] = randn(t, hq, d).half(), randn(t, h, d).half(), randn(t, h, d).half()
        s["q_weight"] = s["k_weight"] = s["cos"] = s["sin"] = None
        if c["norm"]:
            s["q_weight"], s["k_weight"] = (0.3 * randn(d)).exp().half(), (0.3 * randn(d)).exp().half()
        if c["rope"]:
            at = torch.randint(0, 40000, (t, 1), generator=host).to(DEVICE).double()
            angle = at * 1e6 ** (-torch.arange(0, d, 2, device=DEVICE).double() / d)
            s["cos"], s["sin"] = torch.cos(angle).half(), torch.sin(angle).half()
        return s
    rows, kv = _rows_and_keys(c)
    b = c["batch"]
    if c["op"] == "decode":
        live = b - c["idle"]
        s["q"] = randn(b, hq, d).half()
        s["k"], s["v"] = randn(b, h, d).half(), randn(b, h, d).half()
    else:
        cu = torch.zeros(b + 1, dtype=torch.int64)
        cu[1:] = rows.cumsum(0)
        s["q"] = randn(int(cu[-1]), hq, d).half()
        s["rows"], s["most_rows"] = rows.to(DEVICE), int(rows.max())
        s["cu"], s["ctx"] = cu.to(DEVICE, torch.int32), (kv - rows).to(DEVICE, torch.int32)
        s["most_keys"] = int(kv.max())
    each = (kv + page - 1) // page
    used = int(each.sum())
    pages = used + used // 10 + 1
    order = torch.randperm(pages, generator=host)
    table = torch.zeros(b, max(1, int(each.max())), dtype=torch.int64)
    at = torch.arange(table.shape[1]).unsqueeze(0)
    mine = at < each.unsqueeze(1)
    table[mine] = order[:used]
    s["pool"] = _pool(c, pages, g)
    s["table"], s["lens"] = table.to(DEVICE, torch.int32), kv.to(DEVICE, torch.int32)
    if c["op"] == "decode":
        s["last"] = table[torch.arange(b), ((kv - 1) // page).clamp(min=0)][:live].to(DEVICE, torch.int32)
    return s


# ---- one pass ------------------------------------------------------------------------------------------------------------------

def _epilogue(x, weight, s):
    """RMSNorm over each head's row and the rotation of its halves, in float32."""
    y = x.float()
    if weight is not None:
        # the sum in 64 bits: its last bits decide codes that lie next to a border
        y = y * torch.rsqrt(x.double().square().mean(-1, keepdim=True) + 1e-6).float() * weight.float()
    if s["cos"] is not None:
        cos, sin = s["cos"].float().unsqueeze(1), s["sin"].float().unsqueeze(1)
        a, b = y.chunk(2, -1)
        y = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return y


def _keys(s):
    """K and V of every sequence, float32 [B, Hkv, keys, D], padded to the block table's width."""
    c = s["case"]
    b, width = s["table"].shape
    rows = _pages(s["pool"], s["table"].reshape(-1), c).view(b, width * c["page"], 2 * c["hkv"], c["d"]).transpose(1, 2)
    return rows[:, : c["hkv"]].contiguous(), rows[:, c["hkv"]:].contiguous()


def _attend(q, k, v, seen):
    """q [B, Hkv, rows, D], k and v [B, Hkv, keys, D], seen [B, 1, rows, 1]: how many keys a row sees; none gives zeros."""
    x = torch.matmul(q, k.transpose(-1, -2).contiguous()) * (1.0 / math.sqrt(q.shape[-1]))
    x = x.masked_fill(torch.arange(k.shape[2], device=q.device) >= seen, float("-inf"))
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top > float("-inf"), top, torch.zeros_like(top)))
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p, v) / torch.where(total > 0, total, torch.ones_like(total))


def run(s):
    c = s["case"]
    hq, h, d, page = c["hq"], c["hkv"], c["d"], c["page"]
    pool, scale = s["pool"], 1.0 / math.sqrt(d)
    if own:
        from llama_lite_npu_amd import ops

        def held(pages):
            values = torch.empty((pages.numel() * page, 2 * h, d), dtype=torch.float16, device=DEVICE)
            ops.page_dequant(pool, values, pages, None, None, page)
            return values

        if c["op"] == "append":
            if not (c["norm"] or c["rope"]):
                ops.kv_append_quantised(s["k"], s["v"], s["slots"], pool)
                return {"pages": held(s["pages"])}
            ops.qk_norm_rope_append(s["q"], s["k"], s["v"], s["slots"], pool, s["q_weight"], s["k_weight"], s["cos"],
                                    s["sin"], 1e-6)
            return {"q": s["q"], "pages": held(s["pages"])}
        if c["op"] == "prefill":
            return ops.paged_prefill(s["q"], pool, s["table"], s["cu"], s["ctx"], s["most_rows"], scale, page_size=page,
                                     max_kv_len=s["most_keys"])
        if c["append"]:
            out = ops.paged_decode(s["q"], pool, s["table"], s["lens"], scale, page_size=page, k_new=s["k"], v_new=s["v"])
            return {"out": out, "pages": held(s["last"])}
        return ops.paged_decode(s["q"], pool, s["table"], s["lens"], scale, page_size=page)
    if c["op"] == "append":
        if not (c["norm"] or c["rope"]):
            _store(pool, s["slots"], s["k"].float(), s["v"].float(), c)
            return {"pages": _pages(pool, s["pages"], c).half()}
        s["q"].copy_(_epilogue(s["q"], s["q_weight"], s))
        _store(pool, s["slots"], _epilogue(s["k"], s["k_weight"], s), s["v"].float(), c)
        return {"q": s["q"], "pages": _pages(pool, s["pages"], c).half()}
    if c["op"] == "decode":
        b, last = c["batch"], (s["lens"].long() - 1).clamp(min=0)
        if c["append"]:
            slots = s["table"].long().gather(1, (last // page).unsqueeze(1)).squeeze(1) * page + last % page
            _store(pool, torch.where(s["lens"] > 0, slots, -1), s["k"].float(), s["v"].float(), c)
        k, v = _keys(s)
        out = _attend(s["q"].float().view(b, h, hq // h, d), k, v, s["lens"].view(-1, 1, 1, 1)).reshape(b, hq, d).half()
        return {"out": out, "pages": _pages(pool, s["last"], c).half()} if c["append"] else out
    # prefill: rows padded to the longest chunk, the query heads of a kv head next to each other
    b, most, g = c["batch"], s["most_rows"], hq // h
    at = torch.arange(most, device=DEVICE)
    there = at < s["rows"].unsqueeze(1)
    q = torch.zeros(b, most, hq, d, device=DEVICE)
    q[there] = s["q"].float()
    q = q.view(b, most, h, g, d).permute(0, 2, 3, 1, 4).reshape(b, h, g * most, d)
    k, v = _keys(s)
    seen = (s["ctx"].unsqueeze(1) + at + 1).unsqueeze(1).expand(b, g, most).reshape(b, 1, g * most, 1)
    out = _attend(q, k, v, seen).view(b, h, g, most, d).permute(0, 3, 1, 2, 4).reshape(b, most, hq, d)
    return out[there].half()


def work(case):
    c = dict(case)
    hq, h, d = c["hq"], c["hkv"], c["d"]
    row = 2 * h * (d // 2 + 2)                       # a token's K and V in the cache
    if c["op"] == "append":
        t, live = c["tokens"], c["tokens"] - c["idle"]
        pages = live if live <= 256 else -(-live // c["page"])
        fused = c["norm"] or c["rope"]
        read = live * 2 * h * d * 2 + (t * hq * d * 2 if fused else 0) + (t * d * 2 if c["rope"] else 0)
        written = live * row + (t * hq * d * 2 if fused else 0) + pages * c["page"] * 2 * h * d * 2
        return {"bytes": read + written + pages * c["page"] * row, "flops": 0.0}
    rows, keys = _rows_and_keys(c)
    cached, total = int(keys.sum()) * row, int(rows.sum())
    if c["op"] == "decode":
        live = c["batch"] - c["idle"]
        more = live * (2 * h * d * 2 + row + c["page"] * (row + 2 * h * d * 2)) if c["append"] else 0
        return {"bytes": cached + 2 * total * hq * d * 2 + more, "flops": 4.0 * hq * d * int(keys.sum())}
    pairs = int((rows * (keys - rows) + rows * (rows + 1) // 2).sum())
    return {"bytes": cached + 2 * total * hq * d * 2, "flops": 4.0 * hq * d * pairs}


# ---- the definition in 64 bits ---------------------------------------------------------------------------------------------------

def _byte_of(c):
    """For slot t of a block, head and element: the byte its code is in, and whether in its upper half."""
    h, d = c["hkv"], c["d"]
    t, head, e = torch.meshgrid(torch.arange(BLOCK), torch.arange(2 * h), torch.arange(d), indexing="ij")
    # K: nibble e % 8 // 2, four further for odd elements, of the dword of eight elements
    nib_k = e % 8 // 2 + 4 * (e % 2)
    at_k = head * 8 * d + t * d // 2 + e // 8 * 4 + nib_k // 2
    # V: column of d / 16 elements; unit and nibble inside it; a unit is the half-dword t % 2 of pair t / 2 % 2
    wide, units = d // 16, d // 64
    unit, nib_v = e % wide % units, e % wide // units
    at_v = head * 8 * d + t // 4 * 2 * d + e // wide * (d // 8) + (t // 2 % 2 * units + unit) * 4 + t % 2 * 2 + nib_v // 2
    key = head < h
    return torch.where(key, at_k, at_v).to(DEVICE), (torch.where(key, nib_k, nib_v) % 2 == 1).to(DEVICE)


def _values64(pool, tokens, c, where):
    """float64 [n, 2 * Hkv, D]: what the slots `tokens` hold."""
    h, d, at, upper = c["hkv"], c["d"], *where
    blocks = pool.reshape(-1, _block_bytes(c))
    t = tokens % BLOCK
    byte = blocks[(tokens // BLOCK).view(-1, 1, 1), at[t]]
    code = torch.where(upper[t], byte // 16, byte % 16).double()
    word_at = 16 * h * d + 2 * (torch.arange(2 * h, device=DEVICE) * BLOCK + t.unsqueeze(1))
    lo, hi = (blocks[(tokens // BLOCK).unsqueeze(1), word_at + i].long() for i in (0, 1))
    zero, bits = lo % 16, lo - lo % 16 + 256 * hi
    exponent, mantissa = bits // 1024, (bits % 1024).double()
    scale = torch.where(exponent > 0, (1024 + mantissa) * 2.0 ** (exponent.double() - 25), mantissa * 2.0 ** -24)
    return (code - zero.unsqueeze(-1)) * scale.unsqueeze(-1)


def _rounded64(x):
    """float64 rows as the cache holds them."""
    lo, hi = x.amin(-1, keepdim=True).clamp(max=0), x.amax(-1, keepdim=True).clamp(min=0)
    step = (hi - lo) / 15
    exponent = torch.frexp(step).exponent
    unit = torch.ldexp(torch.ones_like(step), torch.clamp(exponent - 7, min=-20))
    s = torch.ceil(step / unit) * unit
    n = x / s.clamp(min=2.0 ** -30)
    z = torch.round(-lo / s.clamp(min=2.0 ** -30))
    return (torch.minimum(torch.maximum(torch.round(n), -z), 15 - z)) * s


def _rows64(x, weight, s):
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + 1e-6) * weight.double()
    if s["cos"] is not None:
        half = x.shape[-1] // 2
        z = torch.complex(x[..., :half], x[..., half:]) * torch.complex(s["cos"].double(), s["sin"].double()).unsqueeze(1)
        x = torch.cat((z.real, z.imag), -1)
    return x


def exact(case, seed):
    c = dict(case)
    s = prepare(case, seed)
    hq, h, d, page = c["hq"], c["hkv"], c["d"], c["page"]
    where = _byte_of(c)
    inside = torch.arange(page, device=DEVICE)

    def pages64(pages, slots, rows):
        """What the pages hold once `rows` are in `slots`."""
        tokens = (pages.long().unsqueeze(1) * page + inside).reshape(-1)
        values = _values64(s["pool"], tokens, c, where)
        place = torch.full((s["pool"].shape[0],), -1, device=DEVICE, dtype=torch.int64)
        place[tokens] = torch.arange(tokens.numel(), device=DEVICE)
        values[place[slots]] = rows
        return values

    if c["op"] == "append":
        live = (s["slots"] >= 0).nonzero().squeeze(-1)
        k, v = s["k"][live], s["v"][live].double()
        part = {**s, **{n: s[n][live] for n in ("cos", "sin") if s[n] is not None}}
        rows = _rounded64(torch.cat((_rows64(k, s["k_weight"], part), v), 1))
        held = pages64(s["pages"], s["slots"][live].long(), rows)
        if not (c["norm"] or c["rope"]):
            return {"pages": held}
        return {"q": _rows64(s["q"], s["q_weight"], s), "pages": held}
    g = hq // h
    lens = s["lens"].tolist()
    new = _rounded64(torch.cat((s["k"], s["v"]), 1).double()) if c["op"] == "decode" and c["append"] else None
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEVICE)
    slots = []
    starts = s["cu"].tolist() if c["op"] == "prefill" else None
    for b, n in enumerate(lens):
        if n == 0:
            continue
        tokens = (s["table"][b].long().unsqueeze(1) * page + inside).reshape(-1)[:n]
        kv = _values64(s["pool"], tokens, c, where)
        if new is not None:
            kv[-1] = new[b]
            slots.append(tokens[-1])
        r0, r1 = (b, b + 1) if starts is None else (starts[b], starts[b + 1])
        last = torch.arange(n - (r1 - r0), n, device=DEVICE).unsqueeze(1)          # the last key each row sees
        hidden = torch.arange(n, device=DEVICE) > last
        q = s["q"][r0:r1].double()
        for head in range(hq):
            x = (q[:, head] @ kv[:, head // g].t()) / math.sqrt(d)
            out[r0:r1, head] = torch.softmax(x.masked_fill(hidden, float("-inf")), -1) @ kv[:, h + head // g]
    if new is not None:
        live = s["lens"].nonzero().squeeze(-1)
        return {"out": out, "pages": pages64(s["last"], torch.stack(slots), new[live])}
    return out
