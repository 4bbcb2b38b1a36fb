"""The operators of a quantised key/value cache, in plain torch and as the framework's kernels, with the sizes they meet.

The cache keeps keys and values in 8 bits (OCP E4M3: a sign, 4 bits of exponent, 3 of fraction, largest value 448) with
one power of two per token and key/value head for the keys and one for the values.  For a head's row x[0 .. D):

    e = the smallest integer in [-117, 119] with max |x| <= 448 * 2^e
    code[d] = x[d] / 2^e rounded to E4M3 (nearest, ties to even), value[d] = code[d] * 2^e, the byte e + 127 is kept

Four operators:

  store    rotate queries and keys of a step's tokens, quantise keys and values, put them into their pages
           (its cases read the rows back, so that the outputs are the values that the codes stand for)
  read     the rows of given tokens out of their pages, as the values they stand for
  decode   attention of one new token per sequence over its pages: out_h = sum_j softmax_j(scale q_h . k_j) v_j
  chunk    causal attention of a run of new tokens per sequence, over the pages that hold what came before and the run itself

Layout of a page (page_size tokens): keys [kv_heads][head_dim / 32][page_size][32], values [kv_heads][head_dim][page_size],
exponent bytes [kv_heads][2][page_size], the keys' before the values'."""

import math

import torch

own = False

DEV = "cuda"

# (query heads, key/value heads, head size): the presets' three, heads without groups, and all queries of one
SMALL, BASE, WIDE, EACH, ONE = (14, 2, 64), (28, 4, 128), (40, 8, 128), (16, 16, 128), (16, 1, 128)


def _case(kind, form, page, seqs, first, last, new=1, window=0):
    """`seqs` sequences that had `first` to `last` tokens in the cache before `new` more of each came."""
    heads, kv, dim = form
    return {"kind": kind, "heads": heads, "kv_heads": kv, "head_dim": dim, "page": page, "seqs": seqs, "first": first,
            "last": last, "new": new, "window": window}


def listed():
    named = {
        # a step of eight decoded tokens of the 7B form writes its keys and values
        "store 8 tokens": _case("store", BASE, 16, 8, 500, 2060),
        # a prompt portion of the default token budget behind what was there before, from a position inside a page
        "store 512 tokens": _case("store", BASE, 16, 1, 1541, 1541, 512),
        # a whole long prompt's portion of the 14B form
        "store 8192 tokens": _case("store", WIDE, 16, 4, 0, 0, 2048),
        # a prefix of one conversation read out of the cache
        "read 333 tokens": _case("read", SMALL, 16, 1, 0, 0, 333),
        # many sequences' prefixes at once
        "read 64 x 2000 tokens": _case("read", BASE, 16, 64, 0, 0, 2000),
        # one short conversation on the smallest form: latency alone
        "decode 1 at 333": _case("decode", SMALL, 16, 1, 333, 333),
        # the default batch
        "decode 8 at 2060": _case("decode", BASE, 16, 8, 2060, 2060),
        # a full batch of unequal lengths
        "decode 64 at 61 to 4000": _case("decode", BASE, 16, 64, 61, 4000),
        # long contexts, larger pages
        "decode 8 at 16000": _case("decode", WIDE, 64, 8, 16000, 16000),
        # a few tokens of a follow-up question in several conversations
        "chunk 4 x 17 at 700 to 1900": _case("chunk", SMALL, 16, 4, 700, 1900, 17),
        # a prompt from its beginning
        "chunk 2048 at 0": _case("chunk", BASE, 16, 1, 0, 0, 2048),
        # the token budget's portion far into a long prompt
        "chunk 512 at 16000": _case("chunk", BASE, 16, 1, 16000, 16000, 512),
    }
    return [dict(c, name=n) for n, c in named.items()]


def _spread(rng, low, high):
    """A whole number of [low, high], evenly over its logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    kind = rng.choice(["store", "read", "decode", "decode", "chunk", "chunk"])
    form = rng.choice([SMALL, BASE, WIDE, EACH, ONE, (32, 8, 128), (24, 8, 96), (9, 3, 64), (16, 4, 32)])
    page = rng.choice([16, 16, 32, 64])
    heads, kv, dim = form
    if kind in ("store", "read"):
        seqs = _spread(rng, 1, 64)
        return _case(kind, form, page, seqs, 0, rng.choice([0, _spread(rng, 1, 16000)]), _spread(rng, 1, 8192 // seqs))
    window = rng.choice([0, 0, 0, _spread(rng, 1, 4096)])
    if kind == "decode":
        seqs = _spread(rng, 1, 128)
        most = min(16000, 128000 * 1024 // (seqs * kv * dim))
        last = _spread(rng, 1, most)
        return _case(kind, form, page, seqs, rng.choice([last, _spread(rng, 1, last)]), last, 1, window)
    seqs = _spread(rng, 1, 8)
    new = _spread(rng, 2, 2048 // seqs)
    last = _spread(rng, 1, max(1, min(16000, 16000 * 512 * 28 * 128 // (seqs * new * heads * dim))))
    return _case(kind, form, page, seqs, rng.choice([last, 0]), last, new, window)


def _starts(case):
    """Tokens that each sequence had before the step, evenly from `first` to `last`."""
    n = case["seqs"]
    return [case["first"] + (case["last"] - case["first"]) * i // max(1, n - 1) if n > 1 else case["last"] for i in range(n)]


def work(case):
    h, kv, d, new = case["heads"], case["kv_heads"], case["head_dim"], case["new"]
    tokens = case["seqs"] * new
    row = 2 * d + 2  # a token's key, value and exponent bytes of one head
    if case["kind"] == "store":  # 16-bit projections in, rotated queries out, codes out and read back as 16-bit values
        return {"bytes": tokens * (2 * (h + 2 * kv) * d + 2 * h * d + kv * 2 * row + 4 * kv * d), "flops": 3 * tokens * (h + 2 * kv) * d}
    if case["kind"] == "read":
        return {"bytes": tokens * kv * (row + 4 * d), "flops": tokens * kv * 2 * d}
    window = case["window"] or 1 << 40
    pairs = read = 0
    for start in _starts(case):
        # the query at position p reads min(p + 1, window) keys
        short = max(0, min(new, window - start))  # queries that the window does not bound
        pairs += short * start + short * (short + 1) // 2 + (new - short) * window if short < new else new * start + new * (new + 1) // 2
        read += min(start + new, window + new - 1)
    return {"bytes": read * kv * row + 2 * 2 * tokens * h * d, "flops": 4 * pairs * h * d}


# ------------------------------------------------------------------ what a user's program has in hand


def _quantise(x):
    """(codes of [..., D] rows, exponent bytes [...])."""
    amax = x.abs().amax(-1)
    m, e = torch.frexp(amax.float())  # amax = m 2^e, 1/2 <= m < 1; 448 = 7/8 * 2^9
    e = (e - 9 + (m > 0.875).int()).clamp(-117, 119)
    e = torch.where(amax == 0, torch.full_like(e, -117), e)
    return torch.ldexp(x, -e[..., None]).float().to(torch.float8_e4m3fn), (e + 127).to(torch.uint8)


def _table(case, gen):
    """Pages of every sequence, in no order, one of the pool left over."""
    lens = [s + case["new"] for s in _starts(case)]
    width = -(-max(lens) // case["page"])
    need = [-(-n // case["page"]) for n in lens]
    order = torch.randperm(sum(need) + 1, generator=gen, device=DEV).to(torch.int32)
    tables = torch.zeros(case["seqs"], width, dtype=torch.int32, device=DEV)
    at = 0
    for i, n in enumerate(need):
        tables[i, :n] = order[at:at + n]
        at += n
    return tables, sum(need) + 1


def prepare(case, seed):
    h, kv, d, ps, new = case["heads"], case["kv_heads"], case["head_dim"], case["page"], case["new"]
    gen = torch.Generator(device=DEV).manual_seed(seed)
    starts = _starts(case)
    tables, pages = _table(case, gen)
    tokens = case["seqs"] * new
    start = torch.tensor(starts, dtype=torch.int32, device=DEV)
    seq = torch.arange(case["seqs"], dtype=torch.int32, device=DEV).repeat_interleave(new)
    s = {
        **case, "starts": starts, "tables": tables, "token_seq": seq,
        "positions": start.repeat_interleave(new) + torch.arange(new, dtype=torch.int32, device=DEV).repeat(case["seqs"]),
        "cu_q": torch.arange(case["seqs"] + 1, dtype=torch.int32, device=DEV) * new, "ctx_lens": start + new,
    }

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=DEV)

    # keys have a few large channels, every token and head a size of its own
    channels = torch.exp(0.5 * normal(kv, d)) if case["kind"] != "store" else torch.exp(0.5 * normal((h + 2 * kv) * d))
    if case["kind"] == "store":
        s["qkv"] = (normal(tokens, (h + 2 * kv) * d) * channels).bfloat16()
        s["inv_freq"] = 1e6 ** (-torch.arange(0, d, 2, device=DEV, dtype=torch.float64) / d)
        s["inv_freq"] = s["inv_freq"].float()
        s["k_pool"] = torch.zeros(pages, kv, d // 32, ps, 32, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)
        s["v_pool"] = torch.zeros(pages, kv, d, ps, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)
        s["scales"] = torch.zeros(pages, kv, 2, ps, dtype=torch.uint8, device=DEV)
        s["q_out"] = torch.empty(tokens, h * d, dtype=torch.bfloat16, device=DEV)
    else:
        k, ke = _quantise(normal(pages, kv, ps, d) * torch.exp(0.3 * normal(pages, kv, ps, 1)) * channels[:, None])
        v, ve = _quantise(normal(pages, kv, ps, d) * torch.exp(0.3 * normal(pages, kv, ps, 1)))
        s["k_pool"] = k.view(torch.uint8).view(pages, kv, ps, d // 32, 32).transpose(2, 3).contiguous().view(torch.float8_e4m3fn)
        s["v_pool"] = v.view(torch.uint8).transpose(2, 3).contiguous().view(torch.float8_e4m3fn)
        s["scales"] = torch.stack([ke, ve], 2).contiguous()
    if case["kind"] in ("store", "read"):
        s["k_out"], s["v_out"] = (torch.empty(tokens, kv * d, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    else:
        s["q"] = normal(tokens, h * d).bfloat16()
        s["out"] = torch.empty(tokens, h * d, dtype=torch.bfloat16, device=DEV)
        # room for the shares of a context that several workgroups take: up to 64 of them, 256 keys or more each
        shares = max(1, min(64, -(-(max(starts) + new) // 256)))
        s["partial"] = torch.empty(min(tokens * h * shares, 1 << 20) * (d + 2), dtype=torch.float32, device=DEV)
    return s


# ------------------------------------------------------------------ one pass


def run(s):
    return _own(s) if own else _plain(s)


def _own(s):
    from shrike_amd.kernels import ops
    from shrike_amd.parts import attention as plans

    h, kv, d, ps = s["heads"], s["kv_heads"], s["head_dim"], s["page"]
    cache = (s["k_pool"], s["v_pool"], s["scales"], ps)
    if s["kind"] in ("store", "read"):
        if s["kind"] == "store":
            ops.rope_kv_store_e4m3(s["qkv"], h, kv, d, d, s["inv_freq"], s["positions"], s["token_seq"], s["tables"], *cache,
                                   q_out=s["q_out"])
        ops.kv_read_e4m3(s["k_out"], s["v_out"], kv, d, s["positions"], s["token_seq"], s["tables"], *cache)
        return (s["q_out"], s["k_out"], s["v_out"]) if s["kind"] == "store" else (s["k_out"], s["v_out"])
    scale, window, reach = d ** -0.5, s["window"] or None, s["window"] or 1 << 40
    if s["kind"] == "decode":
        nsplit = plans.e4m3_decode_splits(s["seqs"], h, kv, d, min(max(s["starts"]) + 1, reach))
        ops.attention_decode_e4m3(s["q"], s["out"], s["seqs"], h, kv, d, s["positions"], s["tables"], *cache, window, scale,
                                  s["partial"], nsplit)
        return s["out"]
    nsplit = plans.e4m3_portion_splits([s["new"]] * s["seqs"], s["starts"], h, kv, d, reach)
    ops.attention_prefill_e4m3(s["q"], s["out"], 0, s["seqs"], h, kv, d, s["cu_q"], s["ctx_lens"], s["tables"], *cache, window,
                               scale, s["partial"], nsplit)
    return s["out"]


def _values(s, page, slot):
    """Keys and values [*page.shape, kv_heads, head_dim] in float32 of the tokens at (page, slot)."""
    kv, d = s["kv_heads"], s["head_dim"]
    k = s["k_pool"].view(torch.uint8)[page, :, :, slot].view(torch.float8_e4m3fn).float().reshape(*page.shape, kv, d)
    v = s["v_pool"].view(torch.uint8)[page, :, :, slot].view(torch.float8_e4m3fn).float()
    e = (s["scales"][page, :, :, slot].int() << 23).view(torch.float32)  # a power of two from its biased exponent
    return k * e[..., 0, None], v * e[..., 1, None]


def _plain(s):
    h, kv, d, ps, new, seqs = s["heads"], s["kv_heads"], s["head_dim"], s["page"], s["new"], s["seqs"]
    pos, seq = s["positions"].long(), s["token_seq"].long()
    if s["kind"] == "read":
        k, v = _values(s, s["tables"][seq, pos // ps].long(), pos % ps)
        return k.reshape(-1, kv * d).bfloat16(), v.reshape(-1, kv * d).bfloat16()
    if s["kind"] == "store":
        x = s["qkv"].float().view(-1, h + 2 * kv, d)
        angle = pos.double()[:, None, None] * s["inv_freq"].double()
        cos, sin = angle.cos().float(), angle.sin().float()
        a, b = x[:, :h + kv, :d // 2], x[:, :h + kv, d // 2:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        code, e = _quantise(torch.cat([turned[:, h:], x[:, h + kv:]], 1))
        back = (code.float() * ((e.int() << 23).view(torch.float32))[..., None]).bfloat16()
        return turned[:, :h].bfloat16().flatten(1), back[:, :kv].flatten(1), back[:, kv:].flatten(1)
    longest = max(s["starts"]) + new
    at = torch.arange(longest, device=DEV)
    k, v = _values(s, s["tables"][:, at // ps].long(), (at % ps).expand(seqs, -1))  # [sequence, key, head, element]
    group = h // kv
    q = s["q"].float().view(seqs, new, kv, group, d).permute(0, 2, 3, 1, 4).reshape(seqs, kv, group * new, d)
    scores = torch.matmul(q, k.permute(0, 2, 3, 1).contiguous()).view(seqs, kv, group, new, longest).mul_(d ** -0.5)
    p = pos.view(seqs, 1, 1, new, 1)
    hidden = (at > p) | (at <= p - s["window"]) if s["window"] else at > p
    scores.masked_fill_(hidden, -math.inf)
    scores -= scores.amax(-1, keepdim=True)
    weights = scores.exp_()
    total = weights.sum(-1, keepdim=True)
    out = torch.matmul(weights.view(seqs, kv, group * new, longest), v.permute(0, 2, 1, 3).contiguous())
    out = out.view(seqs, kv, group, new, d) / total
    return out.permute(0, 3, 1, 2, 4).reshape(seqs * new, h * d).bfloat16()


# ------------------------------------------------------------------ the definition in 64 bits


def _decoded(codes):
    """What E4M3 codes (bytes) stand for, from their bits, in 64 bits."""
    b = codes.to(torch.int64)
    power, fraction = (b >> 3) & 15, (b & 7).double()
    size = torch.where(power == 0, fraction * 2.0 ** -9, (1 + fraction / 8) * torch.pow(2.0, (power - 7).double()))
    return torch.where(b >= 128, -size, size)


def _encoded(x):
    """The values [.., D] rounded to E4M3 times a power of two per row, by the definition, in 64 bits."""
    unit = torch.full_like(x[..., :1], 2.0 ** -117)
    largest = x.abs().amax(-1, keepdim=True)
    for e in range(-116, 120):
        unit = torch.where(largest > 448 * unit, torch.full_like(unit, 2.0 ** e), unit)
    y = x / unit
    # 8 steps from one power of two to the next, from 2^-6 downwards steps of 2^-9
    step = torch.pow(2.0, torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    step = torch.where(y.abs() < step * 8, step / 2, step)  # (where the logarithm has rounded up to a whole number)
    step = torch.where(y.abs() >= step * 16, step * 2, step).clamp(min=2.0 ** -9)
    return torch.round(y / step) * step * unit


def exact(case, seed):
    s = prepare(case, seed)
    h, kv, d, ps, new = case["heads"], case["kv_heads"], case["head_dim"], case["page"], case["new"]
    if case["kind"] == "store":
        x = s["qkv"].double().view(-1, h + 2 * kv, d)
        z = torch.complex(x[:, :h + kv, :d // 2], x[:, :h + kv, d // 2:])
        angle = s["positions"].double()[:, None] * s["inv_freq"].double()
        z = z * torch.polar(torch.ones_like(angle), angle)[:, None]
        turned = torch.cat([z.real, z.imag], -1)
        return turned[:, :h].flatten(1), _encoded(turned[:, h:]).flatten(1), _encoded(x[:, h + kv:]).flatten(1)
    keys, values = [], []  # of each sequence, [token, head, element]
    for i, start in enumerate(s["starts"]):
        page = s["tables"][i, : -(-(start + new) // ps)].long()
        units = torch.pow(2.0, s["scales"][page].double() - 127)
        k = _decoded(s["k_pool"].view(torch.uint8)[page]).transpose(2, 3).reshape(-1, kv, ps, d) * units[:, :, 0, :, None]
        v = _decoded(s["v_pool"].view(torch.uint8)[page]).transpose(2, 3) * units[:, :, 1, :, None]
        keys.append(k.transpose(1, 2).reshape(-1, kv, d)[: start + new])
        values.append(v.transpose(1, 2).reshape(-1, kv, d)[: start + new])
    if case["kind"] == "read":
        return tuple(torch.cat([x[start:].flatten(1) for x, start in zip(y, s["starts"])]) for y in (keys, values))
    q = s["q"].double().view(-1, h, d)
    out = torch.empty_like(q)
    for i, start in enumerate(s["starts"]):
        for head in range(h):
            k, v = keys[i][:, head * kv // h], values[i][:, head * kv // h]
            logits = q[i * new:(i + 1) * new, head] @ k.t() / math.sqrt(d)
            behind = torch.arange(start, start + new, device=DEV)[:, None] - torch.arange(start + new, device=DEV)
            logits[(behind < 0) | (behind >= (case["window"] or start + new))] = -math.inf
            out[i * new:(i + 1) * new, head] = torch.softmax(logits, -1) @ v
    return out.flatten(1)
