"""What the decode step and the prompt of a request with images need beside text attention, as measurable cases.

* ``mrope``: the QKV projection's epilogue for tokens whose position has several axes (time, height, width): per-head RMSNorm of q
  and k, the rotation of their halves by angles that each take one axis' position, and the append of K and V to the paged cache.
  Pair i (elements i and i + D / 2) of a token at positions p_0 .. p_A-1 turns by the angle of table row p_a(i), column i:

      contiguous sections (s_0 .. s_A-1):   a(i) = the section that i lies in
      interleaved sections:                 a(i) = i mod A where that is above 0 and i < A * s_a, else 0

  The cache is fp16, or 8-bit codes with a scale per head (E4M3, or int8 of +-127): code = round(x / scale), value = code * scale.
* ``cross``: the rows of a batch's sequences attend over all of their encoder's states, which lie in pages of their own (fp16, E4M3
  or int8); a sequence without states gets zeros. ``rows`` 0 is the decode step's form, one row a sequence.
* ``sample``: one token per row of logits from a given uniform number. With p_i = exp((x_i - max x) / T), 0 where that is below
  e^-40, tokens ordered by p (ties: the lowest index first), these are kept: the first top_k; of them the shortest run whose mass
  reaches top_p of the first top_k's; of them those of at least min_p times the largest p. The token is the first, by index, at
  which the kept mass exceeds u times all of it; its log-probability is among the kept ones. T = 0 takes the first largest.
"""

import math

import torch

own = False

DEVICE = "cuda:0"
HEADS = ((64, 8, 128), (16, 8, 128), (32, 4, 128), (32, 8, 64))     # query heads, kv heads, head dim
TABLE = 40960                                                       # rows of the cos and sin tables


def _mrope(name, heads, tokens, pool, interleaved, norm=True, page=16, idle=0):
    """``tokens`` rows, the last ``idle`` of which are padding (no slot)."""
    hq, hkv, d = heads
    return {"name": name, "op": "mrope", "hq": hq, "hkv": hkv, "d": d, "tokens": tokens, "pool": pool,
            "interleaved": interleaved, "norm": norm, "page": page, "idle": idle}


def _cross(name, heads, batch, rows, lo, hi, pool="fp16", page=16, none=0, lengths=1):
    """``batch`` sequences of 1..rows rows (0: one each, the decode step's form) over lo..hi states; the last ``none`` of them have
    no states. ``lengths`` seeds how many each has."""
    hq, hkv, d = heads
    return {"name": name, "op": "cross", "hq": hq, "hkv": hkv, "d": d, "batch": batch, "rows": rows, "lo": lo, "hi": hi,
            "pool": pool, "page": page, "none": none, "lengths": lengths}


def _sample(name, batch, vocab, dtype, filters, masked=False):
    """``filters``: which of k (top_k), p (top_p), m (min_p) the requests set; g: some requests are greedy. ``masked``: a grammar
    leaves a part of the vocabulary, the rest is minus infinity."""
    return {"name": name, "op": "sample", "batch": batch, "vocab": vocab, "dtype": dtype, "filters": filters, "masked": masked}


def listed():
    return [
        # one user's decode step on a small model: nothing but latency
        _mrope("mrope-1", HEADS[1], 1, "fp16", False),
        # the serving batch's decode step, four rows of padding among it
        _mrope("mrope-32-int8", HEADS[0], 36, "int8", True, idle=4),
        # an image's tokens on a model without QK norm, narrow heads, larger pages
        _mrope("mrope-image-hd64-fp8", HEADS[3], 1111, "fp8", False, norm=False, page=64),
        # eight prompts' worth of text and image tokens
        _mrope("mrope-prompts", HEADS[0], 10366, "fp16", True),
        # one user's decode step over the states of one clip
        _cross("cross-1", HEADS[1], 1, 0, 1500, 1500),
        # the serving batch's decode step over images of several tiles; two requests have none
        _cross("cross-32", HEADS[0], 32, 0, 400, 6400, none=2),
        # drafts of a few tokens, narrow heads, larger pages, int8
        _cross("cross-drafts-hd64-int8", HEADS[3], 12, 9, 100, 3000, pool="int8", page=64, none=1, lengths=7),
        # prompts about images
        _cross("cross-prompts", HEADS[0], 8, 1024, 1000, 6400, lengths=3),
        # one user's token
        _sample("sample-1", 1, 32000, "fp16", "kp"),
        # the serving batch, every filter in use, greedy requests among it
        _sample("sample-32", 32, 151936, "fp16", "kpmg"),
        # a constrained batch of float32 logits, an odd vocabulary
        _sample("sample-33-masked", 33, 49999, "fp32", "pm", masked=True),
        # a large batch without top_k
        _sample("sample-256", 256, 128000, "bf16", "p"),
    ]


def _between(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("mrope", "cross", "sample"))
    heads = rng.choice(HEADS)
    page = rng.choice((16, 16, 32, 64, 128, 256))
    if op == "mrope":
        tokens = _between(rng, 1, 10000)
        c = _mrope("", heads, tokens, rng.choice(("fp16", "fp8", "int8")), rng.random() < 0.5, rng.random() < 0.7, page,
                   rng.choice((0, 0, min(3, tokens - 1))))
    elif op == "cross":
        hi = _between(rng, 1, 8000)
        rows = rng.choice((0, _between(rng, 1, 1024)))
        most = max(1, min(64 if rows else 256, 8192 // max(1, rows), 1500000 // (hi * heads[1]) if rows == 0 else 64,
                          1500000000 // (heads[0] * max(1, rows) * hi)))
        batch = _between(rng, 1, most)
        c = _cross("", heads, batch, rows, max(1, hi // rng.choice((1, 4, 100))), hi, rng.choice(("fp16", "fp16", "fp8", "int8")),
                   page, rng.choice((0, 0, min(1, batch - 1))), rng.randrange(1000))
    else:
        vocab = _between(rng, 1000, 152000)
        c = _sample("", _between(rng, 1, min(256, 256 * 128000 // vocab)), vocab, rng.choice(("fp16", "bf16", "fp32")),
                    rng.choice(("", "p", "k", "m", "kp", "pm", "kpm", "kpmg")), rng.random() < 0.3)
    del c["name"]
    return c


# ---- inputs --------------------------------------------------------------------------------------------------------------------

def _sections(d):
    """What the axes time, height and width get of the d / 2 pairs."""
    side = 3 * d // 16
    return (d // 2 - 2 * side, side, side)


def _paged(c, slots, g):
    """A pool that has served for a while, and its scales: rows of normal values, or their codes."""
    h, d = c["hkv"], c["d"]
    rows = torch.randn(slots, 2 * h, d, generator=g, device=DEVICE)
    if c["pool"] == "fp16":
        return rows.half(), None
    most = 448.0 if c["pool"] == "fp8" else 127.0
    scales = (torch.rand(2 * h, generator=g, device=DEVICE) * 0.5 + 5.5) / most
    return _codes(rows, scales, c["pool"]), scales


def _lengths(c):
    """Per sequence of a cross case: its rows and its encoder's states."""
    g = torch.Generator().manual_seed(c["lengths"])
    b = c["batch"]
    rows, keys = (torch.randint(lo, hi + 1, (b,), generator=g) for lo, hi in ((1, max(1, c["rows"])), (c["lo"], c["hi"])))
    rows[int(torch.randint(0, b, (1,), generator=g))] = max(1, c["rows"])
    keys[int(torch.randint(0, max(1, b - c["none"]), (1,), generator=g))] = c["hi"]
    if c["none"]:
        keys[b - c["none"]:] = 0
    return rows, keys


def prepare(case, seed):
    c = dict(case)
    g, host = torch.Generator(DEVICE).manual_seed(seed), torch.Generator().manual_seed(seed)
    randn = lambda *shape: torch.randn(shape, generator=g, device=DEVICE)  # noqa: E731
    rand = lambda *shape: torch.rand(shape, generator=g, device=DEVICE)  # noqa: E731
    s = {"case": c}
    if c["op"] == "sample":
        b, v = c["batch"], c["vocab"]
        # a bulk of unlikely tokens, some hundred plausible ones, a few favourites
        x = 2.0 * randn(b, v)
        for n, up in ((300, 5.0), (20, 9.0)):
            x.scatter_add_(1, torch.randint(0, v, (b, n), generator=g, device=DEVICE), up + randn(b, n))
        if c["masked"]:
            x.masked_fill_(rand(b, v) < 0.9, float("-inf"))
            x[:, v // 2] = 1.0
        s["logits"] = x.to({"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}[c["dtype"]])
        s["u"] = rand(b)
        s["temperature"] = 0.6 + 0.8 * rand(b)
        if "g" in c["filters"]:
            s["temperature"][::5] = 0.0
        s["top_k"] = torch.randint(1, 200, (b,), generator=g, device=DEVICE, dtype=torch.int32) if "k" in c["filters"] else None
        s["top_p"] = 0.7 + 0.29 * rand(b) if "p" in c["filters"] else None
        s["min_p"] = 0.2 * rand(b) if "m" in c["filters"] else None
        return s
    hq, h, d, page = c["hq"], c["hkv"], c["d"], c["page"]
    if c["op"] == "mrope":
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
        s["pool"], s["scales"] = _paged(c, pages * page, g)
        s["slots"], s["pages"] = slots.to(DEVICE, torch.int32), order.to(DEVICE, torch.int32)
        s["q"], s["k"], s["v"] = randn(t, hq, d).half(), randn(t, h, d).half(), randn(t, h, d).half()
        s["q_weight"] = s["k_weight"] = None
        if c["norm"]:
            s["q_weight"], s["k_weight"] = (0.3 * randn(d)).exp().half(), (0.3 * randn(d)).exp().half()
        # text and images in turn: an image's tokens share a time and stand on a grid, 32 wide
        i = torch.arange(t)
        image = i // 700 % 2 == 1
        base = int(torch.randint(0, 20000, (1,), generator=host)) + i // 700 * 100
        inside = i % 700
        text = base + inside
        axes = (torch.where(image, base, text), torch.where(image, base + inside // 32, text), torch.where(image, base + inside % 32, text))
        s["positions"] = torch.stack(axes).to(DEVICE)
        angle = torch.arange(TABLE, device=DEVICE).double().unsqueeze(1) * 1e6 ** (-torch.arange(0, d, 2, device=DEVICE).double() / d)
        s["cos"], s["sin"] = torch.cos(angle).half(), torch.sin(angle).half()
        return s
    rows, keys = _lengths(c)
    b = c["batch"]
    each = (keys + page - 1) // page
    used = int(each.sum())
    pages = used + used // 10 + 1
    order = torch.randperm(pages, generator=host)
    table = torch.zeros(b, max(1, int(each.max())), dtype=torch.int64)
    table[torch.arange(table.shape[1]).unsqueeze(0) < each.unsqueeze(1)] = order[:used]
    s["pool"], s["scales"] = _paged(c, pages * page, g)
    s["table"], s["keys"], s["most_keys"] = table.to(DEVICE, torch.int32), keys.to(DEVICE, torch.int32), int(keys.max())
    cu = torch.zeros(b + 1, dtype=torch.int64)
    cu[1:] = rows.cumsum(0)
    s["q"] = randn(int(cu[-1]), hq, d).half()
    s["cu"], s["rows"], s["most_rows"] = cu.to(DEVICE, torch.int32), rows.to(DEVICE), int(rows.max())
    return s


# ---- one pass ------------------------------------------------------------------------------------------------------------------

def _codes(rows, scales, pool):
    """Rows [T, heads, D] in float32 as 8-bit codes."""
    x = rows / scales.view(1, -1, 1)
    if pool == "fp8":
        return x.clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    return torch.round(x).clamp(-127.0, 127.0).to(torch.int8)


def _values(codes, scales):
    """What rows of a pool stand for, in float32."""
    return codes.float() if scales is None else codes.float() * scales.view(-1, 1)


def _turned(x, weight, cos, sin):
    """RMSNorm over each head's row and the rotation of its halves, in float32."""
    y = x.float()
    if weight is not None:
        # the sum in 64 bits: its last bits decide codes that lie next to a border
        y = y * torch.rsqrt(x.double().square().mean(-1, keepdim=True) + 1e-6).float() * weight.float()
    a, b = y.chunk(2, -1)
    return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)


def _axis_of_pair(c):
    i, sections = torch.arange(c["d"] // 2, device=DEVICE), torch.tensor(_sections(c["d"]), device=DEVICE)
    if c["interleaved"]:
        axis = i % 3
        return torch.where(i < 3 * sections[axis], axis, 0)
    return (i.unsqueeze(1) >= sections.cumsum(0)).sum(1)


def _plain_mrope(s):
    c = s["case"]
    h, d, page = c["hkv"], c["d"], c["page"]
    row = s["positions"].clamp(0, TABLE - 1).t()[:, _axis_of_pair(c)]           # [T, D / 2]: rows of the tables
    column = torch.arange(d // 2, device=DEVICE)
    cos, sin = s["cos"][row, column].float().unsqueeze(1), s["sin"][row, column].float().unsqueeze(1)
    s["q"].copy_(_turned(s["q"], s["q_weight"], cos, sin))
    rows = torch.cat((_turned(s["k"], s["k_weight"], cos, sin), s["v"].float()), 1)
    slots = s["slots"].long()
    there = ((slots >= 0) & (slots < s["pool"].shape[0])).nonzero().squeeze(-1)
    if s["scales"] is None:
        s["pool"][slots[there]] = rows[there].half()
        return {"q": s["q"], "pool": s["pool"]}
    # (indexing as bytes: not every type has an indexed write of its own)
    s["pool"].view(torch.uint8)[slots[there]] = _codes(rows[there], s["scales"], c["pool"]).view(torch.uint8)
    held = s["pool"].view(torch.uint8).view(-1, page, 2 * h, d)[s["pages"].long()].view(s["pool"].dtype)
    return {"q": s["q"], "pages": _values(held, s["scales"]).half().view(-1, 2 * h, d)}


def _plain_cross(s):
    c = s["case"]
    hq, h, d, b, most = c["hq"], c["hkv"], c["d"], c["batch"], s["most_rows"]
    g = hq // h
    at = torch.arange(most, device=DEVICE)
    there = at < s["rows"].unsqueeze(1)
    # rows padded to the most of a sequence, the query heads of a kv head next to each other
    q = torch.zeros(b, most, hq, d, device=DEVICE)
    q[there] = s["q"].float()
    q = q.view(b, most, h, g, d).permute(0, 2, 3, 1, 4).reshape(b, h, g * most, d)
    pool = s["pool"] if s["scales"] is None else s["pool"].view(torch.uint8)
    held = pool.view(-1, c["page"], 2 * h, d)[s["table"].long()].view(s["pool"].dtype)       # [B, pages, page, 2 * Hkv, D]
    held = _values(held, s["scales"]).view(b, -1, 2 * h, d).transpose(1, 2)
    k, v = held[:, :h], held[:, h:].contiguous()
    x = torch.matmul(q, k.transpose(-1, -2).contiguous()) * (1.0 / math.sqrt(d))
    x = x.masked_fill(torch.arange(k.shape[2], device=DEVICE) >= s["keys"].view(-1, 1, 1, 1), float("-inf"))
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top > float("-inf"), top, torch.zeros_like(top)))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v) / torch.where(total > 0, total, torch.ones_like(total))
    out = out.view(b, h, g, most, d).permute(0, 3, 1, 2, 4).reshape(b, most, hq, d)
    return out[there].half()


def _plain_sample(s):
    # sums over the whole vocabulary that a token's border is compared with: in 64 bits
    x = s["logits"].float()
    x = torch.where(x.isnan(), float("-inf"), x).clamp(max=torch.finfo(torch.float32).max)
    top, greedy = x.amax(-1, keepdim=True).double(), x.argmax(-1)
    t = s["temperature"].double().unsqueeze(1)
    heat = torch.where(t > 0, t, torch.ones_like(t))
    ordered, order = x.sort(dim=-1, descending=True, stable=True)
    below = ordered.double() - top
    mass = torch.where(below >= -40.0 * heat, torch.exp(below / heat), 0.0)
    keep = mass > 0
    if s["top_k"] is not None:
        keep &= torch.arange(x.shape[1], device=DEVICE) < s["top_k"].unsqueeze(1)
    mass = torch.where(keep, mass, 0.0)
    if s["top_p"] is not None:
        upto = mass.cumsum(-1)
        keep &= upto - mass < s["top_p"].double().unsqueeze(1) * upto[:, -1:]
    if s["min_p"] is not None:
        keep &= below >= heat * torch.log(s["min_p"].double().unsqueeze(1))
    mass = torch.zeros_like(mass).scatter_(1, order, torch.where(keep, mass, 0.0))      # by index again
    upto = mass.cumsum(-1)
    target = s["u"].double().unsqueeze(1) * upto[:, -1:]
    drawn = torch.searchsorted(upto, target, right=True).squeeze(1).clamp(max=x.shape[1] - 1)
    hot = t.squeeze(1) > 0
    share = mass.gather(1, drawn.unsqueeze(1)).squeeze(1) / upto[:, -1]
    return {"tokens": torch.where(hot, drawn, greedy), "logprobs": torch.where(hot, share.log(), 0.0).float()}


def run(s):
    c = s["case"]
    if own:
        from llama_lite_npu_amd import ops

        if c["op"] == "mrope":
            ops.qk_norm_mrope_append(s["q"], s["k"], s["v"], s["slots"], s["pool"], s["positions"], _sections(c["d"]), s["cos"],
                                     s["sin"], s["q_weight"], s["k_weight"], 1e-6, kv_scales=s["scales"],
                                     interleaved=c["interleaved"])
            if s["scales"] is None:
                return {"q": s["q"], "pool": s["pool"]}
            values = torch.empty((s["pages"].numel() * c["page"], 2 * c["hkv"], c["d"]), dtype=torch.float16, device=DEVICE)
            ops.page_dequant(s["pool"], values, s["pages"], None, s["scales"], c["page"])
            return {"q": s["q"], "pages": values}
        if c["op"] == "cross":
            if c["rows"] == 0:
                return ops.paged_cross_attention(s["q"], s["pool"], s["table"], s["keys"], page_size=c["page"],
                                                 kv_scales=s["scales"], max_kv_len=s["most_keys"])
            return ops.paged_cross_attention(s["q"], s["pool"], s["table"], s["keys"], s["cu"], s["most_rows"],
                                             page_size=c["page"], kv_scales=s["scales"], max_kv_len=s["most_keys"])
        tokens, logprobs = ops.sample_tokens(s["logits"], s["u"], s["temperature"], s["top_k"], s["top_p"], s["min_p"],
                                             return_logprobs=True)
        return {"tokens": tokens, "logprobs": logprobs}
    if c["op"] == "mrope":
        return _plain_mrope(s)
    return _plain_cross(s) if c["op"] == "cross" else _plain_sample(s)


def work(case):
    c = dict(case)
    if c["op"] == "sample":
        return {"bytes": c["batch"] * (c["vocab"] * (4 if c["dtype"] == "fp32" else 2) + 32), "flops": 0.0}
    hq, h, d = c["hq"], c["hkv"], c["d"]
    row = 2 * h * d * (2 if c["pool"] == "fp16" else 1)                          # a token's K and V in the cache
    if c["op"] == "mrope":
        t, live = c["tokens"], c["tokens"] - c["idle"]
        read = t * hq * d * 2 + live * 2 * h * d * 2 + t * d * 2 + t * 28        # q, k, v, cos and sin, positions and slots
        written = t * hq * d * 2 + live * row
        if c["pool"] != "fp16":                                                  # and the pages as values
            pages = live if live <= 256 else -(-live // c["page"])
            written += pages * c["page"] * (row + 2 * h * d * 2)
        return {"bytes": read + written, "flops": 0.0}
    rows, keys = _lengths(c)
    return {"bytes": int(keys.sum()) * row + 2 * int(rows.sum()) * hq * d * 2, "flops": 4.0 * hq * d * int((rows * keys).sum())}


# ---- the definition in 64 bits ---------------------------------------------------------------------------------------------------

def _e4m3(x):
    """The nearest E4M3 numbers."""
    x = x.clamp(-448, 448)
    step = torch.ldexp(torch.ones_like(x), torch.frexp(x).exponent.clamp(min=-5) - 4)
    return torch.round(x / step) * step


def exact(case, seed):
    c = dict(case)
    s = prepare(case, seed)
    if c["op"] == "sample":
        tokens, logprobs = [], []
        for r in range(c["batch"]):
            x, t, u = s["logits"][r].double(), float(s["temperature"][r]), float(s["u"][r])
            if t == 0.0:
                tokens.append((x == x.max()).nonzero()[0, 0])
                logprobs.append(x.new_zeros(()))
                continue
            y = (x - x.max()) / t
            y = torch.where(x - x.max() < -40.0 * t, float("-inf"), y)
            n = int((y > float("-inf")).sum())
            k = n if s["top_k"] is None else min(n, int(s["top_k"][r]))
            # the k most likely: all above the k-th value, and the first of those that equal it
            first = torch.argsort(-y, stable=True)[:k]
            w = y[first].exp()
            if s["top_p"] is not None:
                before = torch.cat((w.new_zeros(1), w.cumsum(0)[:-1]))
                w = w[before < float(s["top_p"][r]) * w.sum()]
            if s["min_p"] is not None:
                w = w[w >= float(s["min_p"][r]) * w[0]]
            first = first[: w.numel()].sort().values
            w = y[first].exp()
            i = int((w.cumsum(0) <= u * w.sum()).sum().clamp(max=w.numel() - 1))
            tokens.append(first[i])
            logprobs.append(y[first[i]] - w.sum().log())
        return {"tokens": torch.stack(tokens), "logprobs": torch.stack(logprobs)}
    hq, h, d, page = c["hq"], c["hkv"], c["d"], c["page"]
    scales = torch.ones(2 * h, device=DEVICE) if s["scales"] is None else s["scales"]
    scales = scales.double().view(-1, 1)
    if c["op"] == "mrope":
        places = torch.zeros(c["tokens"], d // 2, dtype=torch.int64, device=DEVICE)
        st, sh, sw = _sections(d)
        columns = torch.arange(d // 2)
        for a in range(3):
            if c["interleaved"]:
                mine = (columns % 3 == a) & (columns < 3 * (st, sh, sw)[a]) if a else columns >= 0
            else:
                mine = (columns >= sum((st, sh, sw)[:a])) & (columns < sum((st, sh, sw)[: a + 1]))
            places[:, mine.to(DEVICE)] = s["positions"][a].unsqueeze(1)
        turn = torch.complex(torch.gather(s["cos"].double(), 0, places), torch.gather(s["sin"].double(), 0, places)).unsqueeze(1)

        def turned(x, weight):
            x = x.double()
            if weight is not None:
                x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / d + 1e-6) * weight.double()
            z = torch.complex(x[..., : d // 2], x[..., d // 2:]) * turn
            return torch.cat((z.real, z.imag), -1)

        live = c["tokens"] - c["idle"]
        rows = torch.cat((turned(s["k"], s["k_weight"]), s["v"].double()), 1)[:live] / scales
        if c["pool"] == "fp8":
            rows = _e4m3(rows)
        elif c["pool"] == "int8":
            rows = torch.round(rows).clamp(-127, 127)
        held = s["pool"].to(torch.float64) if c["pool"] != "fp8" else s["pool"].float().double()
        held = held * scales
        held[s["slots"][:live].long()] = rows * scales
        q = turned(s["q"], s["q_weight"])
        if c["pool"] == "fp16":
            return {"q": q, "pool": held}
        return {"q": q, "pages": held.view(-1, page, 2 * h, d)[s["pages"].long()].view(-1, 2 * h, d)}
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEVICE)
    starts, inside = s["cu"].tolist(), torch.arange(page, device=DEVICE)
    for b, n in enumerate(s["keys"].tolist()):
        if n == 0:
            continue
        slots = (s["table"][b].long().unsqueeze(1) * page + inside).reshape(-1)[:n]
        raw = s["pool"] if s["scales"] is None else s["pool"].view(torch.uint8)
        kv = raw[slots].view(s["pool"].dtype).float().double() * scales
        rows = slice(starts[b], starts[b + 1])
        for head in range(hq):
            x = s["q"][rows, head].double() @ kv[:, head // (hq // h)].t() / math.sqrt(d)
            out[rows, head] = torch.softmax(x, -1) @ kv[:, h + head // (hq // h)]
    return out
