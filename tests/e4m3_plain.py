"""The quantised cache in 64 bits, by its definition, and steps to test it with.

A row x (one head of one token): e is the smallest integer in [-117, 119] with max |x| <= 448 * 2^e, and every element is
the E4M3 number nearest to x / 2^e (ties to even) times 2^e."""

from __future__ import annotations

import math

import torch

E4M3 = torch.float8_e4m3fn


def exponents(x):
    """e of rows [..., D] (float64), by comparison with 448 * 2^e for every e."""
    largest = x.abs().amax(-1)
    e = torch.full(largest.shape, -117, dtype=torch.int64)
    for k in range(-116, 120):
        e[largest > 448 * 2.0 ** (k - 1)] = k
    return e


def rounded(y):
    """y to the nearest E4M3 number, ties to even; beyond 448 (all finite numbers) 448."""
    size = y.abs().clamp(max=448)
    power = torch.floor(torch.log2(size.clamp(min=2.0 ** -6)))
    power = power + (size >= 2.0 ** (power + 1)).double() - ((size < 2.0 ** power) & (power > -6)).double()
    step = 2.0 ** (power - 3)
    return torch.copysign((torch.round(size / step) * step).clamp(max=448), y)


def half_step(y):
    """Half the distance of the E4M3 numbers around y."""
    return 2.0 ** (torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 4)


def quantised(x):
    """(values, exponents) of rows [..., D] in float64."""
    e = exponents(x)
    unit = torch.ldexp(torch.ones_like(x[..., :1]), e[..., None])
    return rounded(x / unit) * unit, e


def rotate(x, positions, inv_freq, rot_dim, adjacent=False, magnitude=1.0):
    """Rows [n, heads, D] in float64 with their first rot_dim elements turned."""
    if not rot_dim:
        return x
    angle = positions.double()[:, None, None] * inv_freq.double()
    c, s = angle.cos() * magnitude, angle.sin() * magnitude
    out = x.clone()
    if adjacent:
        a, b = x[..., 0:rot_dim:2], x[..., 1:rot_dim:2]
        out[..., 0:rot_dim:2], out[..., 1:rot_dim:2] = a * c - b * s, b * c + a * s
    else:
        half = rot_dim // 2
        a, b = x[..., :half], x[..., half:rot_dim]
        out[..., :half], out[..., half:rot_dim] = a * c - b * s, b * c + a * s
    return out


def key_slab(dim):
    return 32 if dim % 32 == 0 else dim


def random_pools(pages, kv, dim, ps, gen, spread=0.5):
    """(k_pool, v_pool, scales, keys, values) on the CPU: codes at random, keys and values [pages, kv, ps, dim] in float64."""
    out = []
    for _ in range(2):
        x = torch.randn(pages, kv, ps, dim, generator=gen, dtype=torch.float64)
        x *= torch.exp(spread * torch.randn(pages, kv, ps, 1, generator=gen, dtype=torch.float64))
        out.append(quantised(x))
    (k, ke), (v, ve) = out
    slab = key_slab(dim)
    k_codes = (k / torch.ldexp(torch.ones_like(k[..., :1]), ke[..., None])).float().to(E4M3).view(torch.uint8)
    v_codes = (v / torch.ldexp(torch.ones_like(v[..., :1]), ve[..., None])).float().to(E4M3).view(torch.uint8)
    k_pool = k_codes.view(pages, kv, ps, dim // slab, slab).transpose(2, 3).contiguous().view(E4M3)
    v_pool = v_codes.transpose(2, 3).contiguous().view(E4M3)
    return k_pool, v_pool, torch.stack([ke + 127, ve + 127], 2).to(torch.uint8).contiguous(), k, v


class Step:
    """A step of sequences with `starts` tokens in the cache and `news` more each, over a pool with pages in no order; `spare` of
    them belong to nobody."""

    def __init__(self, starts, news, ps, seed=0, spare=3):
        gen = torch.Generator().manual_seed(seed)
        self.starts, self.news, self.ps, self.gen = list(starts), list(news), ps, gen
        need = [-(-(a + n) // ps) for a, n in zip(starts, news)]
        self.pages = sum(need) + spare
        order = torch.randperm(self.pages, generator=gen).to(torch.int32)
        self.tables = torch.full((len(need), max(need + [1])), -1, dtype=torch.int32)  # (nobody follows an entry behind the last)
        at = 0
        for i, n in enumerate(need):
            self.tables[i, :n] = order[at:at + n]
            at += n
        self.free = order[at:].long()
        self.positions = torch.cat([torch.arange(a, a + n) for a, n in zip(starts, news)]).to(torch.int32)
        self.token_seq = torch.cat([torch.full((n,), i) for i, n in enumerate(news)]).to(torch.int32)
        self.cu_q = torch.tensor([0] + list(news)).cumsum(0).to(torch.int32)
        self.ctx_lens = torch.tensor([a + n for a, n in zip(starts, news)], dtype=torch.int32)
        self.n = int(self.positions.numel())

    def rows(self, paged, seq, count):
        """The first `count` tokens' rows [count, kv, dim] of a sequence out of [pages, kv, ps, dim]."""
        at = torch.arange(count)
        page = self.tables[seq].long()[at // self.ps]
        return paged[page, :, at % self.ps]


def attention(step, q, keys, values, heads, scale, window=None, chunk=None):
    """(results [n, heads, dim], their weights' mean of |value|, the largest sum |q| |k| scale of a query's scores) in float64."""
    n, kv = step.n, keys.shape[1]
    q = q.double().view(n, heads, -1)
    out, size, reach = torch.zeros_like(q), torch.zeros_like(q), torch.zeros(n, heads, 1, dtype=torch.float64)
    t = 0
    for i, (start, new) in enumerate(zip(step.starts, step.news)):
        if new == 0:
            continue
        k, v = step.rows(keys, i, start + new), step.rows(values, i, start + new)
        for h in range(heads):
            g = h * kv // heads
            s = q[t:t + new, h] @ k[:, g].t() * scale
            behind = torch.arange(start, start + new)[:, None] - torch.arange(start + new)
            hidden = behind < 0
            if window:
                hidden |= behind >= window
            if chunk:
                pos = torch.arange(start, start + new)[:, None]
                hidden |= torch.arange(start + new)[None] // chunk != pos // chunk
            w = torch.softmax(s.masked_fill(hidden, -math.inf), -1)
            out[t:t + new, h] = w @ v[:, g]
            size[t:t + new, h] = w @ v[:, g].abs()
            reach[t:t + new, h, 0] = (q[t:t + new, h].abs() @ k[:, g].abs().t() * scale).masked_fill(hidden, 0).amax(-1)
        t += new
    return out, size, reach


def allowed(out, size, reach, dim, keys, bf16):
    """How far a kernel's results may be from attention()'s.  float32: sums of dim products and of `keys` weights, each step off by at
    most 2^-24 of the sum of the terms' sizes (a score may begin with up to 40 / log2(e), which is added in the same sum: 64 * 2^-24 more at
    most); a score's error moves its weight by as much, and the weights' sum too; the exponential is good to 2^-21.
    bfloat16 besides: the result is rounded (2^-8 of it), and every weight p to p (1 + d), |d| <= 2^-8.  Where the denominator adds up the
    weights before they are rounded, that is at most 2^-8 size; where it adds up the rounded ones, sum p (1 + d) v / sum p (1 + d) - out =
    sum p d (v - out) / sum p (1 + d), at most 2^-8 (size + |out|) (1 + 2^-7)."""
    scores = (dim + 4) * 2.0 ** -24 * reach + 64 * 2.0 ** -24
    fp32 = (2 * scores + 2 * keys * 2.0 ** -24 + 2 * 2.0 ** -21) * size + 2.0 ** -24 * out.abs()
    return fp32 + (2.0 ** -8 * (size + 2 * out.abs()) * (1 + 2.0 ** -7) if bf16 else 0.0)
