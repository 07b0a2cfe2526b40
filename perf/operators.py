"""Attention over a paged key / value cache, as a decoder that generates text runs it around its int8 products: the cases
that the three operators (append, attention of one new token, attention of a prompt) are measured at, their plain forms in
elementary torch operations, and their definition in 64 bits.

A cache holds pages of `page_size` key slots, [pages][kv_heads][page_size][head_dim] for keys and the same for values; a
table row lists a sequence's pages in order. An int8 cache carries one fp32 scale per slot and head (stored = real * scale).
New tokens of a batch are packed rows, sequence b owning rows offsets[b] .. offsets[b + 1]; they are the last ones of its
lengths[b] keys. A row of token i sees the keys up to its own, the last `window` of them where a window is given."""
import math
import random

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i8": torch.int8}
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "i8": 1}


def _case(name, op, act, cache, heads, kv_heads, head_dim, page, batch, past, new=(1, 1), window=0, interleaved=False, lengths=1):
    return {"name": name, "op": op, "act": act, "cache": cache, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "page": page, "batch": batch, "past_low": past[0], "past_high": past[1], "new_low": new[0], "new_high": new[1],
            "window": window, "interleaved": interleaved, "lengths": lengths}


def listed():
    return [
        # one generated token of each of 16 requests goes into an fp16 cache: a few hundred KB, the call's latency is what counts
        _case("append 16 tokens f16", "append", "f16", "f16", 32, 8, 128, 16, 16, (0, 2047)),
        # prompts of four requests, fp32 rows of an int8 QKV product with 12 heads of 64, into an int8 cache
        _case("append prompts f32 to int8", "append", "f32", "i8", 12, 12, 64, 32, 4, (0, 0), (101, 700), lengths=2),
        # a full batch of long prompts, pairs rotated in place (x0 x1, x2 x3, ...)
        _case("append long prompts bf16", "append", "bf16", "bf16", 32, 8, 128, 64, 8, (0, 300), (1500, 2500), interleaved=True, lengths=3),
        # one request, a short context, fp32 activations, every head with keys of its own: latency
        _case("decode one request f32", "decode", "f32", "f16", 12, 12, 64, 16, 1, (127, 127)),
        # an ordinary serving batch, contexts of every length, four query heads to a key head
        _case("decode 32 requests f16", "decode", "f16", "f16", 32, 8, 128, 16, 32, (0, 4095), lengths=4),
        # the same kind of batch twice as large and long, in an int8 cache
        _case("decode 64 requests int8", "decode", "f16", "i8", 32, 8, 128, 32, 64, (1023, 8191), lengths=5),
        # two requests with very long contexts: few rows, a long axis
        _case("decode long contexts bf16", "decode", "bf16", "bf16", 64, 8, 128, 64, 2, (98303, 131071), lengths=6),
        # fp32 activations over an int8 cache, heads of 64, a sliding window
        _case("decode window f32 int8", "decode", "f32", "i8", 16, 2, 64, 16, 24, (0, 6000), window=1024, lengths=7),
        # short prompts of an fp32 model with 12 heads of 64
        _case("prompt short f32", "prompt", "f32", "f16", 12, 12, 64, 16, 4, (0, 0), (5, 128), lengths=8),
        # ragged prompts, some continuing a cached conversation
        _case("prompt ragged f16", "prompt", "f16", "f16", 32, 8, 128, 16, 8, (0, 1500), (33, 1025), lengths=9),
        # a chunk of each of two long documents, over what is cached of them in int8
        _case("prompt chunk int8", "prompt", "f16", "i8", 32, 8, 128, 64, 2, (12001, 16001), (256, 256), lengths=10),
        # one long prompt at once: the most arithmetic
        _case("prompt long bf16", "prompt", "bf16", "bf16", 32, 8, 128, 64, 1, (0, 0), (8192, 8192), lengths=11),
    ]


def _spread(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


def draw(rng):
    most = {op: max((work(c)["bytes"], work(c)["flops"]) for c in listed() if c["op"] == op) for op in ("append", "decode", "prompt")}
    while True:
        op = rng.choice(("append", "decode", "prompt"))
        act, cache = rng.choice((("f32", "f16"), ("f32", "i8"), ("f16", "f16"), ("f16", "i8"), ("bf16", "bf16"), ("bf16", "i8")))
        head_dim = rng.choice((64, 128))
        kv_heads = rng.choice((1, 2, 3, 4, 8, 12))
        heads = kv_heads * rng.choice((1, 2, 3, 4, 7, 8))
        batch = _spread(rng, 1, 64)
        high = _spread(rng, 1, 131071 if op == "decode" and batch <= 2 else 8191)
        new = (1, 1)
        if op == "prompt" or (op == "append" and rng.random() < 0.7):
            new = (1, _spread(rng, 2, 8192 if op == "prompt" else 2500))
        past = (rng.randint(0, high), high) if op != "append" else (0, rng.choice((0, high)))
        c = _case("", op, act, cache, heads, kv_heads, head_dim, rng.choice((8, 16, 32, 64, 128)), batch, past, new,
                  rng.choice((0, 0, _spread(rng, 1, 4096))) if op != "append" else 0, rng.random() < 0.5 and op == "append", rng.randrange(1 << 30))
        del c["name"]
        total, fresh = _lengths(c)
        cells = c["batch"] * heads * max(fresh) * max(total) * (op == "prompt")
        if heads <= 64 and cells <= 32 * 8192 * 8192 and batch * kv_heads * head_dim * max(total) <= 1 << 29 and \
                work(c)["bytes"] <= most[op][0] and work(c)["flops"] <= most[op][1]:
            return c


def _lengths(case):
    """Keys of each sequence with its new tokens, and how many of them are new. Part of the case, not of the seed."""
    r = random.Random(case["lengths"])
    past = [r.randint(case["past_low"], case["past_high"]) for _ in range(case["batch"])]
    new = [r.randint(case["new_low"], case["new_high"]) for _ in range(case["batch"])]
    return [p + n for p, n in zip(past, new)], new


def work(case):
    total, new = _lengths(case)
    h, kv, d, rows = case["heads"], case["kv_heads"], case["head_dim"], sum(new)
    a, c = SIZE[case["act"]], SIZE[case["cache"]]
    slot = 2 * kv * (d * c + (4 if case["cache"] == "i8" else 0))  # bytes of one key and one value of all heads
    lists = 4 * (sum(-(-t // case["page"]) for t in total) + 2 * len(total) + 1)
    if case["op"] == "append":
        angles = len(set().union(*(range(t - n, t) for t, n in zip(total, new))))  # rows of the tables of cosines and sines
        return {"bytes": rows * (2 * h * d * a + 2 * kv * d * a + slot) + angles * d * 4 + lists, "flops": rows * (h + kv) * d * 3}
    w = case["window"] or max(total)
    seen = sum(min(t, n - 1 + w) for t, n in zip(total, new))  # keys that some row of the sequence sees
    pairs = sum(_sum_up_to(t, w) - _sum_up_to(t - n, w) for t, n in zip(total, new))
    return {"bytes": 2 * rows * h * d * a + seen * slot + lists, "flops": 4 * pairs * h * d}


def _sum_up_to(t, w):
    """sum of min(p, w) for p = 1 .. t"""
    m = min(t, w)
    return m * (m + 1) // 2 + (t - m) * w


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    total, new = _lengths(case)
    batch, h, kv, d, page = case["batch"], case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    act, kind, rows = TYPES[case["act"]], TYPES[case["cache"]], sum(new)
    held = [-(-t // page) for t in total]
    pages, wide = sum(held) + 3, max(held)  # a few pages of the pool belong to nobody

    def rand(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32 if dtype == torch.int8 else dtype)

    if kind == torch.int8:
        k, v = (torch.randint(-127, 128, (pages, kv, page, d), generator=g, device="cuda", dtype=torch.int8) for _ in range(2))
        k_scale, v_scale = (40.0 + 20.0 * torch.rand(pages, kv, page, generator=g, device="cuda") for _ in range(2))
    else:
        k, v, k_scale, v_scale = rand(pages, kv, page, d, dtype=kind), rand(pages, kv, page, d, dtype=kind), None, None
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    held_by = torch.tensor(held, device="cuda")
    column = torch.arange(wide, device="cuda")
    at = (torch.cumsum(held_by, 0) - held_by)[:, None] + column
    table = torch.where(column < held_by[:, None], order[at.clamp(max=pages - 1)], 0).contiguous()
    s = {"case": case, "total": total, "new": new, "k": k, "v": v, "k_scale": k_scale, "v_scale": v_scale, "table": table,
         "lengths": torch.tensor(total, dtype=torch.int32, device="cuda"),
         "offsets": torch.tensor([0] + [sum(new[: b + 1]) for b in range(batch)], dtype=torch.int32, device="cuda")}
    if case["op"] == "append":
        s["qkv"] = rand(rows, (h + 2 * kv) * d, dtype=act)  # one row of the merged projection: all query heads, keys, values
        angle = torch.arange(max(total), device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, d, 2, device="cuda", dtype=torch.float64) / d)
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
    else:
        s["q"] = rand(rows, h, d, dtype=act)
    if own:
        s["plan"] = _plan(s)
    return s


def _views(s):
    c = s["case"]
    h, kv, d = c["heads"], c["kv_heads"], c["head_dim"]
    q, k, v = s["qkv"].view(-1, h + 2 * kv, d).split((h, kv, kv), 1)
    return q, k, v


def _plan(s):
    """What a serving loop keeps: the handles of its cache and batch, and the attention's workspace."""
    from bolt_amd import host_paged
    c = s["case"]
    cache = host_paged.PagedKvCache(s["k"], s["v"], s["k_scale"], s["v_scale"])
    single = c["new_high"] == 1
    batch = host_paged.PagedBatch(s["table"], s["lengths"], None if single else s["offsets"], sum(s["new"]))
    if c["op"] == "append":
        return cache, batch, host_paged.Rotary(s["cos"], s["sin"], c["interleaved"])
    return cache, batch, host_paged.paged_attention_workspace(cache, batch, c["heads"])


def _own(s):
    from bolt_amd import host_paged
    c, (cache, batch, kept) = s["case"], s["plan"]
    if c["op"] == "append":
        q, k, v = _views(s)
        out = host_paged.kv_cache_append(cache, batch, k, v, q, kept)
        return {"q": out, "k": _real(s["k"], s["k_scale"]), "v": _real(s["v"], s["v_scale"])}
    attend = host_paged.paged_attention_decode if c["op"] == "decode" else host_paged.paged_attention_prompt
    return attend(cache, batch, s["q"], window=c["window"], workspace=kept)


def run(s):
    if own:
        return _own(s)
    return _plain_append(s) if s["case"]["op"] == "append" else _plain_attention(s)


def _real(stored, scale):
    """What a cache holds: its own values, or those that its 8-bit numbers stand for."""
    return stored if scale is None else stored.float() * (1.0 / scale)[..., None]


def _owners(s):
    """Of every packed row: its sequence, and its position there."""
    rows = sum(s["new"])
    row = torch.arange(rows, device="cuda")
    seq = torch.searchsorted(s["offsets"][1:].long(), row, right=True)
    return seq, s["lengths"][seq].long() - (s["offsets"][seq + 1].long() - row)


def _rotated(x, cos, sin, interleaved):
    half = x.shape[-1] // 2
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :half], x[..., half:])
    a, b = a * cos - b * sin, b * cos + a * sin
    return torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)


def _plain_append(s):
    c = s["case"]
    q, k, v = (x.float() for x in _views(s))
    seq, pos = _owners(s)
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
    q, k = _rotated(q, cos, sin, c["interleaved"]), _rotated(k, cos, sin, c["interleaved"])
    page, slot = s["table"][seq, pos // c["page"]].long(), pos % c["page"]
    for x, name in ((k, "k"), (v, "v")):
        if c["cache"] == "i8":
            top = x.abs().amax(-1)
            scale = torch.where(top > 0, 127.0 / top, torch.ones_like(top))
            s[name + "_scale"][page, :, slot] = scale
            x = (x * scale[..., None]).round().clamp(-127, 127)
        s[name][page, :, slot] = x.to(s[name].dtype)
    return {"q": q.to(TYPES[c["act"]]), "k": _real(s["k"], s["k_scale"]), "v": _real(s["v"], s["v_scale"])}


def _gathered(s, name):
    """[batch, kv_heads, keys, head_dim] in fp32, as many keys as the longest sequence's pages have"""
    x, scale = s[name][s["table"].long()].float(), s[name + "_scale"]
    if scale is not None:
        x = x * (1.0 / scale[s["table"].long()])[..., None]
    x = x.transpose(1, 2)
    return x.reshape(*x.shape[:2], -1, x.shape[-1])


def _plain_attention(s):
    c = s["case"]
    h, kv, d, batch = c["heads"], c["kv_heads"], c["head_dim"], c["batch"]
    group, rows, most = h // kv, sum(s["new"]), max(s["new"])
    k, v = _gathered(s, "k"), _gathered(s, "v")
    i = torch.arange(most, device="cuda")
    start, count = s["offsets"][:-1].long(), (s["offsets"][1:] - s["offsets"][:-1]).long()
    q = s["q"][(start[:, None] + i).clamp(max=rows - 1)].float()                     # [batch, most, heads, d]
    q = q.view(batch, most, kv, group, d).permute(0, 2, 3, 1, 4).reshape(batch, kv, group * most, d)
    score = torch.matmul(q, k.transpose(-1, -2).contiguous()).mul_(1.0 / math.sqrt(d)).view(batch, kv, group, most, -1)
    pos = s["lengths"].long()[:, None] - count[:, None] + i                            # [batch, most]
    key = torch.arange(k.shape[2], device="cuda")
    sees = key <= pos[..., None]
    if c["window"]:
        sees &= key > pos[..., None] - c["window"]
    score.masked_fill_(~sees[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = score.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(batch, kv, group * most, -1), v).view(batch, kv, group, most, d) / total
    out = out.permute(0, 3, 1, 2, 4).reshape(batch, most, h, d)
    seq, at = _owners(s)
    return out[seq, at - (s["lengths"][seq].long() - count[seq])].to(TYPES[c["act"]])


def exact(case, seed):
    s = prepare(case, seed)
    total, new, page = s["total"], s["new"], case["page"]
    h, kv, d = case["heads"], case["kv_heads"], case["head_dim"]
    table = s["table"].tolist()
    if case["op"] == "append":
        q, k, v = (x.double() for x in _views(s))
        where = [(b, total[b] - new[b] + i) for b in range(case["batch"]) for i in range(new[b])]
        pos = torch.tensor([p for _, p in where], device="cuda")
        turn = torch.complex(s["cos"].double(), s["sin"].double())[pos][:, None]
        two = (2, d // 2) if not case["interleaved"] else (d // 2, 2)
        apart = -2 if not case["interleaved"] else -1

        def rotate(x):
            x = x.unflatten(-1, two)
            z = torch.complex(x.select(apart, 0).contiguous(), x.select(apart, 1).contiguous()) * turn
            return torch.stack((z.real, z.imag), apart).flatten(-2)
        if case["cache"] == "i8":  # which of two neighbours an 8-bit number is, a value next to a border leaves open
            return {"q": rotate(q), "k": None, "v": None}
        keys, values = s["k"].double(), s["v"].double()
        into = torch.tensor([table[b][p // page] for b, p in where], device="cuda")
        keys[into, :, pos % page], values[into, :, pos % page] = rotate(k), v
        return {"q": rotate(q), "k": keys, "v": values}
    out, row = torch.empty_like(s["q"], dtype=torch.float64), 0
    for b in range(case["batch"]):
        mine = torch.tensor(table[b][: -(-total[b] // page)], device="cuda")
        pos = torch.arange(total[b] - new[b], total[b], device="cuda")[:, None]
        key = torch.arange(total[b], device="cuda")
        hidden = (key > pos) | (key <= pos - (case["window"] or total[b]))
        for j in range(kv):
            k, v = (s[n][mine, j].double().reshape(-1, d) for n in ("k", "v"))
            if case["cache"] == "i8":
                k, v = (x / s[n + "_scale"][mine, j].double().reshape(-1, 1) for x, n in ((k, "k"), (v, "v")))
            for i in range(j * h // kv, (j + 1) * h // kv):
                weight = s["q"][row:row + new[b], i].double() @ k[: total[b]].t() / math.sqrt(d)
                weight = torch.softmax(weight.masked_fill(hidden, -math.inf), -1)
                out[row:row + new[b], i] = weight @ v[: total[b]]
        row += new[b]
    return out
