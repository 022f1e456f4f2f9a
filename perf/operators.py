"""The serving-step operators of gpud_amd.diag.serving, as measurable cases.

Four operators of one token step of a served language model: the product with
4-bit weights, the append to an 8-bit paged key/value cache, the attention
over that cache, and the log probabilities of given tokens. `run` computes
each in its plain form from elementary torch operations, or, where `own` is
true, through the framework's entry points.

Storage that both forms read (made by `prepare`, in torch):

* 4-bit codes: uint8 [ceil(N/16), ceil(K/128), 64, 16]. Tile (n, b) holds rows
  16n..16n+15 and columns 128b..128b+127; lane 16g+r holds row r, and its dword
  j the 8 columns 32j + 8g + e, e = 2 (i mod 4) + i // 4 in nibble i.
  Scales [ceil(N/16), ceil(K/G), 16] in x's type, zeros likewise in uint8.
* cache: keys float8_e4m3fn [pages, heads, page, D], values [pages, heads, D,
  page] (a token's values are a column), scales float32 [pages, heads].
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
F8 = torch.float8_e4m3fn
F8_MAX = 448.0
SCALE_FLOOR_EXP = -64
INF = float("inf")


def listed():
    return [
        # one user's token through a square projection: latency counts
        dict(name="w4 1x4096x4096", op="w4", m=1, n=4096, k=4096, group=128, zeros=False, dtype="bf16"),
        # a small decode batch through an odd-sized projection, groups of 64 with zero points
        dict(name="w4 5x5000x5000", op="w4", m=5, n=5000, k=5000, group=64, zeros=True, dtype="fp16"),
        # a decode batch through a large up projection
        dict(name="w4 16x28672x8192", op="w4", m=16, n=28672, k=8192, group=128, zeros=True, dtype="bf16"),
        # the largest batch that decodes together, finest groups
        dict(name="w4 64x16384x8192", op="w4", m=64, n=16384, k=8192, group=32, zeros=False, dtype="bf16"),
        # a decode step's append: one token for each of 256 sequences, pages partly filled
        dict(name="append step 256", op="append", batch=256, new_lo=1, new_hi=1, old_lo=0, old_hi=2000,
             heads=8, dim=128, page=64, dtype="bf16"),
        # prompts and chunks of prompts of several users, written at once
        dict(name="append prompts 24k", op="append", batch=12, new_lo=1, new_hi=4096, old_lo=0, old_hi=900,
             heads=8, dim=128, page=64, dtype="bf16"),
        # one user's step on a short context: latency counts
        dict(name="attn 1x500", op="attn", batch=1, q_lo=0, q_hi=0, len_lo=500, len_hi=500, idle=0,
             q_heads=16, kv_heads=2, dim=64, page=16, window=0, dtype="fp16"),
        # a decode step of a mixed batch, idle slots among it
        dict(name="attn 32x4k mixed", op="attn", batch=32, q_lo=0, q_hi=0, len_lo=1, len_hi=4100, idle=2,
             q_heads=32, kv_heads=8, dim=128, page=64, window=0, dtype="bf16"),
        # the largest decode step: 64 long contexts
        dict(name="attn 64x16k", op="attn", batch=64, q_lo=0, q_hi=0, len_lo=8000, len_hi=16384, idle=0,
             q_heads=64, kv_heads=8, dim=128, page=64, window=0, dtype="bf16"),
        # chunks of prompts among single tokens, against what was cached before
        dict(name="attn chunks 8x4k", op="attn", batch=8, q_lo=1, q_hi=256, len_lo=700, len_hi=4100, idle=0,
             q_heads=32, kv_heads=8, dim=128, page=32, window=0, dtype="bf16"),
        # one token's distribution over a vocabulary, with its alternatives: latency counts
        dict(name="logprobs 1x32000", op="logprobs", rows=1, vocab=32000, top=20, masked=0.0, dtype="fp32"),
        # a scored batch over a large, odd vocabulary with forbidden tokens
        dict(name="logprobs 2048x130001", op="logprobs", rows=2048, vocab=130001, top=5, masked=0.05, dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["w4", "append", "attn", "logprobs"])
    if op == "w4":
        group = rng.choice([32, 64, 128])
        m, n = _log_int(rng, 1, 64), _log_int(rng, 16, 28672)
        k = min(_log_int(rng, 128, 16384), max(128, 235_000_000 // n))
        k = rng.choice([k, -(-k // group) * group, -(-k // 8) * 8])
        return dict(op=op, m=m, n=n, k=k, group=group, zeros=rng.random() < 0.5, dtype=rng.choice(["bf16", "fp16"]))
    heads, dim = rng.choice([1, 2, 4, 8]), rng.choice([64, 80, 128, 256])
    page, dtype = rng.choice([16, 32, 64, 128]), rng.choice(["bf16", "fp16"])
    if op == "append":
        batch = _log_int(rng, 1, 256)
        most = max(1, min(4096, 49152 // batch))
        hi = _log_int(rng, 1, most)
        return dict(op=op, batch=batch, new_lo=1, new_hi=hi, old_lo=0, old_hi=_log_int(rng, 1, 2000),
                    heads=heads, dim=min(dim, 128), page=page, dtype=dtype)
    if op == "attn":
        group = rng.choice([1, 3, 4, 8, 16])
        batch = _log_int(rng, 1, 64)
        hi = min(_log_int(rng, 16, 16384), 3_000_000_000 // (batch * heads * dim * 4))
        q_hi = rng.choice([0, 0, 0, _log_int(rng, 1, 256)])
        q_hi = min(q_hi, hi, max(1, 250_000_000 // (batch * heads * group * hi)))
        return dict(op=op, batch=batch, q_lo=min(1, q_hi), q_hi=q_hi, len_lo=max(1, q_hi, hi // rng.choice([1, 2, 50])), len_hi=hi,
                    idle=rng.choice([0, 1]) if batch > 3 and not q_hi else 0, q_heads=heads * group, kv_heads=heads, dim=dim,
                    page=page, window=rng.choice([0, 0, _log_int(rng, 16, 4096)]), dtype=dtype)
    vocab = _log_int(rng, 200, 200000)
    rows = min(_log_int(rng, 1, 2048), 260_000_000 // vocab)
    return dict(op=op, rows=rows, vocab=vocab, top=rng.choice([0, 1, 5, 20, 50]), masked=rng.choice([0.0, 0.05, 0.9]),
                dtype=rng.choice(["bf16", "fp16", "fp32"]))


def _spread(lo, hi, count):
    """`count` whole numbers spread evenly from lo to hi, so that their sum is known without the seed."""
    return [hi if count == 1 else lo + (hi - lo) * i // (count - 1) for i in range(count)]


def _lengths(case):
    """(tokens held before, query or new tokens) of each sequence, before the seed orders them."""
    b = case["batch"]
    if case["op"] == "append":
        new = _spread(case["new_lo"], case["new_hi"], b)
        old = _spread(case["old_lo"], case["old_hi"], b)
        return old[::-1], new
    lens = _spread(case["len_lo"], case["len_hi"], b)
    q = _spread(case["q_lo"], case["q_hi"], b) if case["q_hi"] else [1] * b
    for i in range(case["idle"]):
        lens[i * (b // 2)] = 0
    return lens, q


def work(case):
    op = case["op"]
    if op == "w4":
        m, n, k = case["m"], case["n"], case["k"]
        groups = -(-k // case["group"])
        size = n * k / 2 + n * groups * (3 if case["zeros"] else 2) + 2 * m * k + 2 * m * n
        return {"bytes": size, "flops": 2 * m * n * k}
    if op == "append":
        _, new = _lengths(case)
        values = 2 * sum(new) * case["heads"] * case["dim"]
        return {"bytes": values * 2 + values, "flops": 3 * values}
    if op == "attn":
        lens, q = _lengths(case)
        h, d, w = case["kv_heads"], case["dim"], case["window"]
        keys = pairs = 0
        for length, n in zip(lens, q):
            keys += min(length, w + n - 1) if w else length
            for i in range(min(n, length)):
                seen = length - n + i + 1
                pairs += min(seen, w) if w else seen
        rows = sum(q) * case["q_heads"]
        return {"bytes": keys * h * (2 * d + 8 / case["page"]) + rows * (4 * d + 4), "flops": 4 * pairs * case["q_heads"] * d}
    size = {"bf16": 2, "fp16": 2, "fp32": 4}[case["dtype"]]
    cells = case["rows"] * case["vocab"]
    return {"bytes": cells * size + case["rows"] * (24 + 12 * case["top"]), "flops": 6 * cells}


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _pages(case, g, lens):
    """A shuffled page table over pages enough for `lens` tokens, as a long-running allocator leaves it."""
    page, b = case["page"], case["batch"]
    need = [-(-n // page) for n in lens]
    total = sum(need) + 3
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(b, max(need + [1]), dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    return table, total


def _cache(case, g, pages):
    """Pages full of codes of normal values at scales of several sizes, with what earlier owners left."""
    h, d, page = case["kv_heads"] if case["op"] == "attn" else case["heads"], case["dim"], case["page"]

    def codes(*shape):
        flat = torch.empty(shape, dtype=F8, device="cuda")
        for i in range(0, shape[0], 256):
            part = torch.randn((min(256, shape[0] - i),) + shape[1:], generator=g, device="cuda")
            flat[i:i + 256] = (part * 90).clamp(-F8_MAX, F8_MAX).to(F8)
        return flat

    def scales():
        e = torch.randint(-8, -4, (pages, h), generator=g, device="cuda")
        return torch.exp2(e.float())

    return codes(pages, h, page, d), codes(pages, h, d, page), scales(), scales()


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    dtype = DTYPES[case["dtype"]]
    s = {"case": case}
    if op == "w4":
        m, n, k = case["m"], case["n"], case["k"]
        tiles, blocks, groups = -(-n // 16), -(-k // 128), -(-k // case["group"])
        s["x"] = torch.randn(m, k, generator=g, device="cuda").to(dtype)
        s["codes"] = torch.randint(0, 256, (tiles, blocks, 64, 16), generator=g, device="cuda", dtype=torch.uint8)
        s["scales"] = (torch.rand(tiles, groups, 16, generator=g, device="cuda") * 0.01 + 0.002).to(dtype)
        s["zeros"] = torch.randint(5, 11, (tiles, groups, 16), generator=g, device="cuda", dtype=torch.uint8) if case["zeros"] else None
        return s
    if op == "logprobs":
        r, v = case["rows"], case["vocab"]
        x = torch.randn(r, v, generator=g, device="cuda") * 2.5
        if case["masked"]:
            x.masked_fill_(torch.rand(r, v, generator=g, device="cuda") < case["masked"], -INF)
        targets = torch.randint(0, v, (r,), generator=g, device="cuda")
        targets[(torch.rand(r, generator=g, device="cuda") < 0.5)] %= max(1, v // 100)
        x.scatter_(1, targets[:, None], torch.randn(r, 1, generator=g, device="cuda") * 4 + 4)  # given tokens are allowed ones
        s["logits"], s["targets"] = x.to(dtype), targets
        return s
    order = torch.randperm(case["batch"], generator=g, device="cuda").tolist()
    a, n = _lengths(case)
    a, n = [a[i] for i in order], [n[i] for i in order]
    total = [x + y for x, y in zip(a, n)] if op == "append" else a
    s["table"], pages = _pages(case, g, total)
    s["k"], s["v"], s["k_scale"], s["v_scale"] = _cache(case, g, pages)
    s["lens"] = torch.tensor(total, dtype=torch.int32, device="cuda")
    starts = [0]
    for x in n:
        starts.append(starts[-1] + x)
    single = op == "attn" and case["q_hi"] == 0 or op == "append" and case["new_hi"] == 1
    s["starts"] = None if single else torch.tensor(starts, dtype=torch.int32, device="cuda")
    s["most"], s["longest"] = max(n), max(total)
    h, d = case["heads"] if op == "append" else case["kv_heads"], case["dim"]
    if op == "append":  # new keys and values lie in one fused projection's output
        both = torch.randn(starts[-1], 2, h, d, generator=g, device="cuda")
        both *= torch.exp2(torch.randint(-2, 3, (starts[-1], 2, h, 1), generator=g, device="cuda").float())
        both = both.to(dtype)
        s["k_new"], s["v_new"] = both[:, 0], both[:, 1]
        return s
    s["q"] = torch.randn(starts[-1], case["q_heads"], d, generator=g, device="cuda").to(dtype)
    # behind a sequence's last token its page holds what an earlier owner left, codes for NaN among it
    page = case["page"]
    for i, length in enumerate(total):
        if length % page:
            p = int(s["table"][i, length // page])
            junk = torch.randint(0, 256, (h, page - length % page, d), generator=g, device="cuda", dtype=torch.uint8)
            junk[:, ::2, ::3] = 0x7F
            s["k"][p, :, length % page:] = junk.view(F8)
            s["v"][p, :, :, length % page:] = junk.transpose(1, 2).view(F8)
    return s


def _unpack(codes, n, k):
    """uint8 tiles -> float32 codes [n, k]."""
    tiles, blocks = codes.shape[:2]
    nibbles = torch.stack((codes & 15, codes >> 4), -1)  # [tiles, blocks, lane, byte, low/high]
    nibbles = nibbles.view(tiles, blocks, 4, 16, 4, 2, 4)  # g, row, j, i // 4, i mod 4
    return nibbles.permute(0, 3, 1, 4, 2, 6, 5).reshape(tiles * 16, blocks * 128)[:n, :k].float()


def _plain_w4(s):
    c = s["case"]
    n, k, group = c["n"], c["k"], c["group"]
    q = _unpack(s["codes"], n, k)

    def spread(t):
        return t.float().permute(0, 2, 1).reshape(-1, t.shape[1])[:n].repeat_interleave(group, 1)[:, :k]

    w = (q - (spread(s["zeros"]) if s["zeros"] is not None else 8.0)) * spread(s["scales"])
    return (s["x"].float() @ w.t()).to(s["x"].dtype)


def _rows_of(s):
    """Of each new or query token: its sequence and its position in it."""
    lens = s["lens"].long()
    if s["starts"] is None:
        return torch.arange(len(lens), device="cuda"), lens - 1
    starts = s["starts"].long()
    t = torch.arange(s["q"].shape[0] if "q" in s else s["k_new"].shape[0], device="cuda")
    seq = torch.searchsorted(starts, t, right=True) - 1
    return seq, lens[seq] - (starts[seq + 1] - t)


def _scale_for(amax):
    """The smallest power of two that brings amax within 448, not under 2^-64."""
    bits = amax.contiguous().view(torch.int32)
    e = ((bits + 0x1FFFFF) >> 23) - 127 - 8
    return torch.exp2(e.clamp_min(SCALE_FLOOR_EXP).float())


def _plain_append(s):
    c = s["case"]
    page, heads = c["page"], c["heads"]
    seq, pos = _rows_of(s)
    lens, b = s["lens"].long(), len(s["lens"])
    new = torch.zeros(b, dtype=torch.long, device="cuda").index_add_(0, seq, torch.ones_like(seq))
    first = lens - new
    # each sequence's touched pages; entries past its last one repeat it
    span = (s["most"] + page - 2) // page + 1
    blocks = first[:, None] // page + torch.arange(span, device="cuda")
    blocks = torch.minimum(blocks, (lens[:, None] - 1) // page)
    pages = s["table"].long().gather(1, blocks)  # [b, span]
    slot = (pos // page - first[seq] // page)
    for cache, scale, x in ((s["k"], s["k_scale"], s["k_new"]), (s["v"], s["v_scale"], s["v_new"])):
        x = x.float()
        amax = torch.zeros(b * span, heads, device="cuda")
        amax.scatter_reduce_(0, (seq * span + slot)[:, None].expand(-1, heads), x.abs().amax(-1), "amax")
        need = _scale_for(amax).view(b, span, heads)
        held = (first[:, None] > blocks * page)[..., None]  # tokens before the new ones stay in the page
        old = scale[pages]
        now = torch.where(held, torch.maximum(old, need), need)
        last = (lens - 1) // page - first // page
        now = now.gather(1, torch.minimum(torch.arange(span, device="cuda"), last[:, None])[..., None].expand(-1, -1, heads))
        ratio = torch.where(held, old / now, torch.ones_like(old))
        flat = cache.view(torch.uint8)
        body = (flat[pages].view(F8).float() * ratio[..., None, None]).clamp(-F8_MAX, F8_MAX)
        flat[pages] = body.to(F8).view(torch.uint8)
        code = (x / now[seq, slot][..., None]).clamp(-F8_MAX, F8_MAX).to(F8)
        at = pages[seq, slot]
        if cache is s["k"]:
            flat[at, :, pos % page] = code.view(torch.uint8)
        else:
            flat[at, :, :, pos % page] = code.view(torch.uint8)
        scale[pages] = now
    return {"k": s["k"], "v": s["v"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def _plain_attn(s):
    c = s["case"]
    b, hk, d, page, dtype = c["batch"], c["kv_heads"], c["dim"], c["page"], s["q"].dtype
    group, most = c["q_heads"] // hk, s["most"]
    seq, pos = _rows_of(s)
    table = s["table"].long()
    span = table.shape[1] * page
    lens = s["lens"].long()
    at = torch.arange(span, device="cuda")
    live = at < lens[:, None]  # [b, span]
    k8, v8 = (s[x].view(torch.uint8)[table].view(F8) for x in ("k", "v"))
    k = (k8.float() * s["k_scale"][table][..., None, None]).permute(0, 2, 1, 3, 4).reshape(b, hk, span, d)
    v = (v8.float() * s["v_scale"][table][..., None, None]).permute(0, 2, 1, 4, 3).reshape(b, hk, span, d)
    k = k.masked_fill_(~live[:, None, :, None], 0.0)
    v = v.masked_fill_(~live[:, None, :, None], 0.0)
    # query tokens in rows of `most` for each sequence
    place = torch.arange(len(seq), device="cuda") - (s["starts"].long()[seq] if s["starts"] is not None else seq)
    q = torch.zeros(b, most, hk, group, d, device="cuda")
    q[seq, place] = s["q"].float().view(-1, hk, group, d)
    at_pos = torch.full((b, most), -1, dtype=torch.long, device="cuda")
    at_pos[seq, place] = pos
    seen = at <= at_pos[..., None]  # [b, most, span]
    if c["window"]:
        seen &= at > at_pos[..., None] - c["window"]
    q = q.permute(0, 2, 1, 3, 4).reshape(b, hk, most * group, d)
    score = (q @ k.transpose(2, 3)) * d ** -0.5
    seen = seen[:, None, :, None].expand(-1, hk, -1, group, -1).reshape(b, hk, most * group, span)
    score = score.masked_fill_(~seen, -INF)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -INF, 0.0, top))
    total = p.sum(-1, keepdim=True)
    out = torch.where(total > 0, (p @ v) / total, 0.0)
    lse = (torch.log(total) + top).squeeze(-1)
    out = out.view(b, hk, most, group, d).permute(0, 2, 1, 3, 4)[seq, place].reshape(-1, c["q_heads"], d)
    lse = lse.view(b, hk, most, group).permute(0, 2, 1, 3)[seq, place].reshape(-1, c["q_heads"])
    return {"out": out.to(dtype), "lse": lse}


def _plain_logprobs(s):
    x, t, top = s["logits"].float(), s["targets"], s["case"]["top"]
    v = x.shape[1]
    xt = x.gather(1, t[:, None])
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - m)
    total = e.sum(-1, keepdim=True)
    norm = m + torch.log(total)
    entropy = (torch.log(total) - torch.where(e > 0, e * (x - m), 0.0).sum(-1, keepdim=True) / total).squeeze(1)
    out = {"logprob": (xt - norm).squeeze(1), "entropy": entropy, "rank": (x > xt).sum(-1)}
    if top:
        # whole-number keys: the value's order above, the lower index first below
        bits = (x + 0.0).view(torch.int32)
        key = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).long() << 32
        key |= v - 1 - torch.arange(v, device="cuda")
        best = torch.topk(key, top, dim=1).values
        ids = v - 1 - (best & 0xFFFFFFFF)
        out["top_ids"], out["top_logprobs"] = ids, x.gather(1, ids) - norm
    return out


def run(state):
    s = state
    c = s["case"]
    op = c["op"]
    if own:
        from gpud_amd.diag import serving

        if op == "w4":
            return serving.w4_matmul(s["x"], s["codes"], s["scales"], s["zeros"], out_features=c["n"], group_size=c["group"])
        if op == "append":
            serving.cache_append(s["k_new"], s["v_new"], s["k"], s["v"], s["k_scale"], s["v_scale"], s["table"], s["lens"], s["starts"])
            return {"k": s["k"], "v": s["v"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
        if op == "attn":
            out, lse = serving.cache_attention(s["q"], s["k"], s["v"], s["k_scale"], s["v_scale"], s["table"], s["lens"], s["starts"],
                                               max_seq_len=s["longest"], window=c["window"] or None)
            return {"out": out, "lse": lse}
        r = serving.token_logprobs(s["logits"], s["targets"], c["top"])
        out = {"logprob": r.logprob, "entropy": r.entropy, "rank": r.rank}
        if c["top"]:
            out["top_ids"], out["top_logprobs"] = r.top_ids, r.top_logprobs
        return out
    return {"w4": _plain_w4, "append": _plain_append, "attn": _plain_attn, "logprobs": _plain_logprobs}[op](s)


def exact(case, seed):
    s = prepare(case, seed)
    return {"w4": _exact_w4, "append": _exact_append, "attn": _exact_attn, "logprobs": _exact_logprobs}[case["op"]](s)


def _exact_w4(s):
    c = s["case"]
    n, k, group = c["n"], c["k"], c["group"]
    x = s["x"].double()
    y = torch.zeros(c["m"], n, dtype=torch.float64, device="cuda")
    column = torch.arange(k, device="cuda")
    block, inside = column // 128, column % 128
    j, g, e = inside // 32, inside % 32 // 8, inside % 8
    nibble = e // 2 + 4 * (e % 2)
    row = torch.arange(n, device="cuda")
    for i in range(0, n, 2048):
        r = row[i:i + 2048, None]
        byte = s["codes"][r // 16, block, g * 16 + r % 16, j * 4 + nibble // 2]
        q = (byte >> (4 * (nibble % 2)).to(torch.uint8)) & 15
        z = s["zeros"][r // 16, column // group, r % 16].double() if c["zeros"] else 8.0
        w = (q.double() - z) * s["scales"][r // 16, column // group, r % 16].double()
        y[:, i:i + 2048] = x @ w.t()
    return y


def _exact_append(s):
    c = s["case"]
    page, lens = c["page"], s["lens"].tolist()
    starts = s["starts"].tolist() if s["starts"] is not None else list(range(c["batch"] + 1))
    if sum(-(-(y - x) // page) + 1 for x, y in zip(starts, starts[1:])) > 6000:
        return None
    table = s["table"].tolist()
    out = {}
    for name, x in (("k", s["k_new"]), ("v", s["v_new"])):
        cache = s[name] if name == "k" else s[name].transpose(2, 3)  # [page, head, token, dim]
        scales = s[name + "_scale"]
        values, now = cache.double(), scales.double()
        for b, length in enumerate(lens):
            first = length - (starts[b + 1] - starts[b])
            for block in range(first // page, (length - 1) // page + 1):
                lo, hi = max(first, block * page), min(length, block * page + page)
                p = table[b][block]
                fresh = x[starts[b] + lo - first:starts[b] + hi - first].double().transpose(0, 1)  # [head, token, dim]
                need = torch.log2(fresh.abs().amax((1, 2)).clamp_min(1e-300) / F8_MAX).ceil().clamp_min(SCALE_FLOOR_EXP)
                e = need
                if lo > block * page:
                    e = torch.maximum(need, torch.log2(now[p]))
                    values[p] *= torch.exp2(torch.log2(now[p]) - e)[:, None, None]
                now[p] = torch.exp2(e)
                values[p, :, lo - block * page:hi - block * page] = fresh / now[p][:, None, None]
        out[name] = values if name == "k" else values.transpose(2, 3)
        out[name + "_scale"] = now
    return out


def _exact_attn(s):
    c = s["case"]
    page, hk, d = c["page"], c["kv_heads"], c["dim"]
    group = c["q_heads"] // hk
    lens, table = s["lens"].tolist(), s["table"].tolist()
    starts = s["starts"].tolist() if s["starts"] is not None else list(range(c["batch"] + 1))
    out = torch.zeros(starts[-1], c["q_heads"], d, dtype=torch.float64, device="cuda")
    lse = torch.full((starts[-1], c["q_heads"]), -INF, dtype=torch.float64, device="cuda")
    for b, length in enumerate(lens):
        count = starts[b + 1] - starts[b]
        if not length or not count:
            continue
        ids = torch.tensor(table[b][:-(-length // page)], device="cuda")
        k = s["k"][ids].double() * s["k_scale"][ids].double()[:, :, None, None]
        v = s["v"][ids].double() * s["v_scale"][ids].double()[:, :, None, None]
        k = k.transpose(0, 1).reshape(hk, -1, d)[:, :length]
        v = v.permute(1, 0, 3, 2).reshape(hk, -1, d)[:, :length]
        j = torch.arange(length, device="cuda")
        for i in range(0, count, 32):
            rows = slice(starts[b] + i, starts[b] + min(count, i + 32))
            p = torch.arange(length - count + i, length - count + min(count, i + 32), device="cuda")[:, None]
            hidden = j > p
            if c["window"]:
                hidden |= j <= p - c["window"]
            q = s["q"][rows].double().view(-1, hk, group, d).permute(1, 2, 0, 3)  # [hk, group, row, d]
            score = torch.matmul(q.reshape(hk, -1, d), k.transpose(1, 2)) / math.sqrt(d)
            score = score.view(hk, group, -1, length).masked_fill(hidden, -INF)
            total = torch.logsumexp(score, -1, keepdim=True)
            got = torch.matmul(torch.exp(score - total).view(hk, -1, length), v).view(hk, group, -1, d)
            out[rows] = got.permute(2, 0, 1, 3).reshape(-1, c["q_heads"], d)
            lse[rows] = total.squeeze(-1).permute(2, 0, 1).reshape(-1, c["q_heads"])
    return {"out": out, "lse": lse}


def _exact_logprobs(s):
    c = s["case"]
    parts = []
    for i in range(0, c["rows"], 256):
        x, t = s["logits"][i:i + 256].double(), s["targets"][i:i + 256]
        p = torch.log_softmax(x, -1)
        part = {"logprob": p.gather(1, t[:, None]).squeeze(1), "entropy": torch.special.entr(p.exp()).sum(-1)}
        if c["top"]:
            part["top_logprobs"] = p.sort(dim=1, descending=True).values[:, :c["top"]]
        parts.append(part)
    out = {k: torch.cat([p[k] for p in parts]) for k in parts[0]}
    out["rank"] = None
    if c["top"]:
        out["top_ids"] = None
    return out
