"""Cases of the decode-time operators around a 4-bit key/value cache.

Three operators, each in a plain form of elementary torch operations (32 bits,
rounded once at the end) and, with `own` set, as calls of openquant_b200:

  rotary     rotary positions on [tokens, heads, head_dim]: half or interleaved
             pairs, all or the first rotary_dim of a head, or the inverse
             rotation (the gradient)
  append     rotates the queries and keys of a step's tokens and writes keys
             and values into a paged cache as 4-bit integers with one scale per
             group; what the cache then holds is read back as values
  attention  queries against that cache: single tokens, a few tokens per
             sequence, chunks of a prompt and mixtures of them

Cache layout: codes uint8 [pages, kv_heads, page, head_dim / 2] (element 2i in
the low nibble, two's complement), scales fp16 [pages, kv_heads, page,
head_dim / group].  A group's scale is max|x| / 7 rounded to 8 significant bits
(bf16) and kept as fp16, at most 9344, 1 where that is 0; its codes are
round(x / scale) limited to -7..7.  Token j of sequence b is in page
page_table[b, j // page] at j % page.  lengths[b] counts a sequence's tokens
with the step's own, which are its last starts[b + 1] - starts[b].
"""
import math

import torch

own = False

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


# ------------------------------------------------------------------ cases --


def listed():
    return [
        # One decode step of 32 requests: queries of a 32-head model (latency).
        dict(name="rotary_step", op="rotary", dtype="fp16", tokens=32, heads=32, dim=128, rotary=128,
             interleaved=False, inverse=False),
        # The queries of a long prompt, 64 heads.
        dict(name="rotary_prompt", op="rotary", dtype="bf16", tokens=8192, heads=64, dim=128, rotary=128,
             interleaved=False, inverse=False),
        # Gradient of a partial, interleaved rotation; an odd token count.
        dict(name="rotary_gradient_part", op="rotary", dtype="fp32", tokens=2049, heads=40, dim=128, rotary=64,
             interleaved=True, inverse=True),
        # One decode step of 64 requests, 64 query heads on 8 key heads.
        dict(name="append_step", op="append", dtype="bf16", heads=64, kv_heads=8, dim=128, group=32, page=16,
             batch=64, length=4096, least=100, tokens=1, fewest=1, interleaved=False),
        # Ragged prompts of a 32-head model going into the cache.
        dict(name="append_prompts", op="append", dtype="fp16", heads=32, kv_heads=32, dim=128, group=64, page=64,
             batch=7, length=2048, least=129, tokens=2048, fewest=129, interleaved=False),
        # One request, one token, a short context: what a chat's first answer tokens cost (latency).
        dict(name="step_one_request", op="attention", dtype="fp16", heads=32, kv_heads=32, dim=128, group=32,
             page=16, batch=1, length=1000, least=1000, tokens=1, fewest=1, window=0),
        # A serving batch of ragged contexts, 64 query heads on 8 key heads.
        dict(name="step_batch", op="attention", dtype="bf16", heads=64, kv_heads=8, dim=128, group=32, page=64,
             batch=64, length=8192, least=333, tokens=1, fewest=1, window=0),
        # Two long documents, one token each.
        dict(name="step_long", op="attention", dtype="bf16", heads=64, kv_heads=8, dim=128, group=64, page=128,
             batch=2, length=131071, least=100003, tokens=1, fewest=1, window=0),
        # Checking 5 drafted tokens per request; 64-wide heads and a sliding window.
        dict(name="verify_window", op="attention", dtype="fp16", heads=24, kv_heads=8, dim=64, group=32, page=16,
             batch=24, length=6001, least=17, tokens=5, fewest=2, window=2048),
        # A chunk of a long prompt over what is cached of it: the largest.
        dict(name="prompt_chunk", op="attention", dtype="bf16", heads=64, kv_heads=8, dim=128, group=32, page=64,
             batch=1, length=32768, least=32768, tokens=4096, fewest=4096, window=0),
        # Whole ragged prompts, one key head per query head.
        dict(name="prompts_ragged", op="attention", dtype="fp16", heads=32, kv_heads=32, dim=128, group=128, page=64,
             batch=5, length=2500, least=77, tokens=2500, fewest=77, window=0),
        # A step that mixes decoding requests with chunks of prompts.
        dict(name="mixed_step", op="attention", dtype="bf16", heads=40, kv_heads=8, dim=128, group=32, page=32,
             batch=20, length=4096, least=600, tokens=500, fewest=1, window=0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        op = rng.choice(["rotary", "append", "attention", "attention", "attention"])
        dim = rng.choice([64, 128, 128])
        if op == "rotary":
            case = dict(op=op, dtype=rng.choice(["fp16", "bf16", "fp32"]), tokens=_log(rng, 1, 16384),
                        heads=_log(rng, 1, 64), dim=dim, rotary=rng.choice([dim, dim // 2, dim // 4]),
                        interleaved=rng.random() < 0.5, inverse=rng.random() < 0.3)
        else:
            kv_heads = rng.choice([1, 2, 4, 8, 8, 32])
            heads = kv_heads * (1 if kv_heads == 32 else rng.choice([1, 3, 4, 5, 7, 8, 16]))
            case = dict(op=op, dtype=rng.choice(["fp16", "bf16"]), heads=heads, kv_heads=kv_heads, dim=dim,
                        group=rng.choice([g for g in (32, 64, 128) if g <= dim]), page=rng.choice([16, 32, 64, 128]))
            batch = _log(rng, 1, 128)
            if op == "append":
                tokens = rng.choice([1, _log(rng, 2, 4096)])
                length = tokens + rng.choice([0, _log(rng, 1, 4096)])
                case.update(batch=batch, length=length, least=max(1, tokens), tokens=tokens,
                            fewest=max(1, tokens // 3), interleaved=rng.random() < 0.5)
            else:
                tokens = rng.choice([1, 1, _log(rng, 2, 8), _log(rng, 9, 4096)])
                length = tokens + _log(rng, 1, 65536)
                case.update(batch=batch, length=length, least=max(tokens, length // rng.choice([1, 2, 10])),
                            tokens=tokens, fewest=max(1, tokens // rng.choice([1, 4])),
                            window=rng.choice([0, 0, 0, _log(rng, 16, 8192)]))
        # The plain form holds all scores and the unpacked cache at once.
        if op == "attention":
            scores = case["batch"] * case["heads"] * case["tokens"] * case["length"]
            unpacked = case["batch"] * case["length"] * case["kv_heads"] * case["dim"]
            if scores > 9e9 or unpacked > 1.2e9:
                continue
        if op == "append" and case["batch"] * case["tokens"] * case["heads"] * case["dim"] > 1.5e8:
            continue
        if _cost(case) <= most:
            return case


def _spread(lo, hi, count):
    """`count` whole numbers over lo..hi, hi among them, in an order of no kind."""
    vals = [hi - (hi - lo) * i // max(1, count - 1) for i in range(count)]
    return [vals[(i * 7 + 3) % count] for i in range(count)] if count % 7 else vals


def _shape(case):
    """(lengths, token counts) of a case's sequences."""
    lengths = _spread(case["least"], case["length"], case["batch"])
    counts = _spread(case["fewest"], case["tokens"], case["batch"])
    return lengths, [min(n, t) for n, t in zip(lengths, counts)]


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "rotary":
        values = case["tokens"] * case["heads"] * case["dim"]
        table = case["tokens"] * (case["rotary"] * 4 + 4)
        return {"bytes": 2 * values * size + table, "flops": 3 * case["tokens"] * case["heads"] * case["rotary"]}
    lengths, counts = _shape(case)
    total = sum(counts)
    token = 2 * case["kv_heads"] * (case["dim"] // 2 + 2 * case["dim"] // case["group"])  # bytes of a cached token
    if case["op"] == "append":
        q, kv = total * case["heads"] * case["dim"], 2 * total * case["kv_heads"] * case["dim"]
        # q in and out, k and v in, the cache's bytes out and, to be read back, in, the values out
        return {"bytes": 2 * q * size + kv * size + 2 * total * token + kv * 2 + total * case["dim"] * 4,
                "flops": 3 * (q + kv // 2) + 6 * kv}
    pairs = seen = 0
    for n, t in zip(lengths, counts):
        w = case["window"] or n
        first = n - t  # cached before the step
        pairs += sum(min(w, first + i + 1) for i in range(t))
        seen += n - max(0, first + 1 - w)
    return {"bytes": 2 * total * case["heads"] * case["dim"] * size + seen * token,
            "flops": 4 * pairs * case["heads"] * case["dim"]}


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 6.5e12, w["flops"] / 1.6e15)


# ----------------------------------------------------------------- inputs --


def _normal(gen, *shape):
    return torch.randn(*shape, device="cuda", generator=gen)


def _table(rows, dim):
    """cos | sin of position * 10000^(-2i / dim), fp32 [rows, dim]."""
    freq = 10000.0 ** (-torch.arange(0, dim, 2, device="cuda", dtype=torch.float64) / dim)
    angle = torch.arange(rows, device="cuda", dtype=torch.float64)[:, None] * freq
    return torch.cat([angle.cos(), angle.sin()], dim=1).float()


def _quantise(x, group):
    """Codes (packed) and scales of x [..., dim] in fp32."""
    parts = x.unflatten(-1, (-1, group))
    seven = torch.full((), 7.0, device=x.device)
    scale = (parts.abs().amax(-1) / seven).bfloat16().half().clamp(max=9344.0)
    scale = torch.where(scale == 0, torch.ones_like(scale), scale)
    codes = (parts / scale.float()[..., None]).round().clamp(-7, 7).to(torch.int8).flatten(-2)
    low, high = codes[..., 0::2] & 15, codes[..., 1::2] & 15
    return (low | (high << 4)).view(torch.uint8), scale


def _values(codes, scales, dim):
    """What packed codes and their scales stand for, fp32 [..., dim]."""
    b = codes.to(torch.int32)
    n = torch.stack([b & 15, b >> 4], dim=-1).flatten(-2)
    n = torch.where(n > 7, n - 16, n).float()
    return (n.unflatten(-1, (scales.shape[-1], -1)) * scales.float()[..., None]).flatten(-2)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, st = TYPES[case["dtype"]], {"case": case}
    if case["op"] == "rotary":
        rows = 32768
        st["x"] = _normal(gen, case["tokens"], case["heads"], case["dim"]).to(dtype)
        st["table"] = _table(rows, case["rotary"])
        st["positions"] = torch.randint(0, rows, (case["tokens"],), device="cuda", generator=gen, dtype=torch.int32)
        return st
    lengths, counts = _shape(case)
    total, dim, kv, page = sum(counts), case["dim"], case["kv_heads"], case["page"]
    slots = -(-case["length"] // page)
    pages = sum(-(-n // page) for n in lengths) + 3
    order = torch.randperm(pages, device="cuda", generator=gen).to(torch.int32)
    st["page_table"] = torch.zeros(len(lengths), slots, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(lengths):
        used = -(-n // page)
        st["page_table"][b, :used] = order[at:at + used]
        at += used
    st["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    starts = [0]
    for t in counts:
        starts.append(starts[-1] + t)
    st["starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda") if max(counts) > 1 else None
    st["most"] = max(counts)
    # Queries and keys of a trained model: a few channels are much larger than the rest.
    channel = torch.ones(dim, device="cuda")
    channel[torch.randint(0, dim, (4,), device="cuda", generator=gen)] = 5.0
    st["q"] = _normal(gen, total, case["heads"], dim).to(dtype)
    if case["op"] == "append":
        st["k"] = (_normal(gen, total, kv, dim) * channel).to(dtype)
        st["v"] = _normal(gen, total, kv, dim).to(dtype)
        st["table"] = _table(case["length"], dim)
        for x in "kv":
            st[x + "_codes"] = torch.zeros(pages, kv, page, dim // 2, dtype=torch.uint8, device="cuda")
            st[x + "_scales"] = torch.zeros(pages, kv, page, dim // case["group"], dtype=torch.float16, device="cuda")
    else:
        st["k_codes"], st["k_scales"] = _quantise(_normal(gen, pages, kv, page, dim) * channel, case["group"])
        st["v_codes"], st["v_scales"] = _quantise(_normal(gen, pages, kv, page, dim), case["group"])
    if own:
        from openquant_b200.kv_cache import Int4KVCache, KVBatch

        st["cache"] = Int4KVCache(st["k_codes"], st["k_scales"], st["v_codes"], st["v_scales"])
        st["batch"] = KVBatch(st["page_table"], st["lengths"], st["starts"], max_tokens=st["most"])
    return st


# ------------------------------------------------------------ plain forms --


def _rotate(x, table, positions, interleaved, inverse=False):
    """x [tokens, heads, dim] turned by its tokens' angles, fp32."""
    x, turn = x.float(), table[positions.long()][:, None]
    half = table.shape[1] // 2
    cos, sin = turn[..., :half], turn[..., half:]
    if inverse:
        sin = -sin
    out = x.clone()
    first = slice(0, 2 * half, 2) if interleaved else slice(0, half)
    second = slice(1, 2 * half, 2) if interleaved else slice(half, 2 * half)
    a, b = x[..., first], x[..., second]
    out[..., first] = a * cos - b * sin
    out[..., second] = b * cos + a * sin
    return out


def _owner(st, total):
    """(sequence, its place among the step's tokens, its position) of each of the step's tokens."""
    t = torch.arange(total, device="cuda")
    if st["starts"] is None:
        return t, torch.zeros_like(t), st["lengths"].long() - 1
    starts = st["starts"].long()
    seq = torch.searchsorted(starts[1:].contiguous(), t, right=True)
    i = t - starts[seq]
    return seq, i, st["lengths"].long()[seq] - (starts[seq + 1] - starts[seq]) + i


def _plain_append(st):
    case, dim = st["case"], st["case"]["dim"]
    seq, _, pos = _owner(st, st["q"].shape[0])
    q = _rotate(st["q"], st["table"], pos, case["interleaved"]).to(st["q"].dtype)
    page, slot = st["page_table"].long()[seq, pos // case["page"]], pos % case["page"]
    st["k_codes"][page, :, slot], st["k_scales"][page, :, slot] = _quantise(
        _rotate(st["k"], st["table"], pos, case["interleaved"]), case["group"])
    st["v_codes"][page, :, slot], st["v_scales"][page, :, slot] = _quantise(st["v"].float(), case["group"])
    k = _values(st["k_codes"][page, :, slot], st["k_scales"][page, :, slot], dim).half()
    v = _values(st["v_codes"][page, :, slot], st["v_scales"][page, :, slot], dim).half()
    return q, k, v


def _plain_attention(st):
    case, q = st["case"], st["q"]
    dim, kv, length, most = case["dim"], case["kv_heads"], case["length"], st["most"]
    each = case["heads"] // kv
    j = torch.arange(length, device="cuda")
    page, slot = st["page_table"].long()[:, j // case["page"]], j % case["page"]
    k = _values(st["k_codes"][page, :, slot], st["k_scales"][page, :, slot], dim).transpose(1, 2)
    v = _values(st["v_codes"][page, :, slot], st["v_scales"][page, :, slot], dim).transpose(1, 2)
    lengths = st["lengths"].long()
    starts = st["starts"].long() if st["starts"] is not None else torch.arange(len(lengths) + 1, device="cuda")
    count = starts[1:] - starts[:-1]
    i = torch.arange(most, device="cuda")
    rows = q[(starts[:-1, None] + i).clamp(max=q.shape[0] - 1)].float()  # [batch, most, heads, dim]
    rows = rows.unflatten(2, (kv, each)).permute(0, 2, 1, 3, 4).flatten(2, 3)
    s = torch.matmul(rows, k.transpose(2, 3)).mul_(1 / math.sqrt(dim))
    pos = (lengths - count)[:, None] + i
    seen = (j <= pos[..., None]) & (i < count[:, None])[..., None]
    if case["window"]:
        seen &= j > pos[..., None] - case["window"]
    seen = seen[:, None, :, None].expand(-1, -1, -1, each, -1).flatten(2, 3)
    s.masked_fill_(~seen, -math.inf)
    top = s.amax(-1, keepdim=True)
    s.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    total = s.sum(-1, keepdim=True)
    o = torch.matmul(s, v) / torch.where(total == 0, torch.ones_like(total), total)
    o = o.unflatten(2, (most, each)).permute(0, 2, 1, 3, 4).flatten(2, 3)  # [batch, most, heads, dim]
    seq, i, _ = _owner(st, q.shape[0])
    return o[seq, i].to(q.dtype)


def run(st):
    case = st["case"]
    if case["op"] == "rotary":
        if own:
            from openquant_b200.kv_cache import rotary

            return rotary(st["x"], st["table"], st["positions"], interleaved=case["interleaved"],
                          inverse=case["inverse"])
        return _rotate(st["x"], st["table"], st["positions"], case["interleaved"], case["inverse"]).to(st["x"].dtype)
    if case["op"] == "append":
        if own:
            q = st["cache"].append(st["k"], st["v"], st["batch"], q=st["q"], table=st["table"],
                                   interleaved=case["interleaved"])
            return (q, *st["cache"].read(st["batch"], st["q"].shape[0]))
        return _plain_append(st)
    if own:
        return st["cache"].attention(st["q"], st["batch"], window=case["window"])
    return _plain_attention(st)


# ----------------------------------------------------------------- 64 bits --


def _exact_rotation(x, table, positions, interleaved, sign):
    """The rotation as a product of complex numbers."""
    half = table.shape[1] // 2
    t = table[positions.long()].double()
    turn = torch.complex(t[:, :half], sign * t[:, half:])[:, None]
    y = x.double().clone()
    part = y[..., :2 * half]
    if interleaved:
        z = torch.view_as_complex(part.unflatten(-1, (half, 2)).contiguous()) * turn
        y[..., :2 * half] = torch.view_as_real(z).flatten(-2)
    else:
        z = torch.complex(part[..., :half].contiguous(), part[..., half:].contiguous()) * turn
        y[..., :2 * half] = torch.cat([z.real, z.imag], dim=-1)
    return y


def _exact_cached(x, group):
    """x as the cache holds it: each group on its grid of 15 values."""
    out = torch.empty_like(x)
    for g in range(0, x.shape[-1], group):
        part = x[..., g:g + group]
        step = (part.abs().max(-1, keepdim=True).values / 7).to(torch.bfloat16).half().double().clamp(max=9344)
        step[step == 0] = 1
        out[..., g:g + group] = torch.round(part / step).clamp(-7, 7) * step
    return out


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "rotary":
        return _exact_rotation(st["x"], st["table"], st["positions"], case["interleaved"],
                               -1.0 if case["inverse"] else 1.0)
    lengths, counts = _shape(case)
    if case["op"] == "append":
        pos = torch.cat([torch.arange(n - t, n, device="cuda") for n, t in zip(lengths, counts)])
        turned = [_exact_rotation(st[x], st["table"], pos, case["interleaved"], 1.0) for x in "qk"]
        return turned[0], _exact_cached(turned[1], case["group"]), _exact_cached(st["v"].double(), case["group"])
    signed = torch.tensor([c - 16 if c > 7 else c for c in range(16)], dtype=torch.float64, device="cuda")
    outs, at, each = [], 0, case["heads"] // case["kv_heads"]
    for b, (n, t) in enumerate(zip(lengths, counts)):
        where = st["page_table"][b, :-(-n // case["page"])].long()
        rows = torch.arange(n - t, n, device="cuda")[:, None]
        cols = torch.arange(n, device="cuda")[None]
        hidden = cols > rows
        if case["window"]:
            hidden = hidden | (cols <= rows - case["window"])
        heads = []
        for h in range(case["kv_heads"]):
            held = []
            for x in "kv":
                codes = st[x + "_codes"][where, h].flatten(0, 1)[:n].long()
                scales = st[x + "_scales"][where, h].flatten(0, 1)[:n].double()
                both = torch.stack([signed[codes % 16], signed[codes // 16]], 2).flatten(1)
                held.append(both * scales.repeat_interleave(case["group"], 1))
            for m in range(each):
                for r in range(0, t, 1024):  # a few rows at a time: scores in 64 bits are large
                    part = slice(r, min(t, r + 1024))
                    s = st["q"][at + part.start:at + part.stop, h * each + m].double() @ held[0].T / math.sqrt(case["dim"])
                    heads.append(torch.softmax(s.masked_fill(hidden[part], -math.inf), 1) @ held[1])
        whole = torch.cat(heads).view(case["heads"], t, case["dim"])
        outs.append(whole.transpose(0, 1))
        at += t
    return torch.cat(outs)
