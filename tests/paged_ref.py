"""64-bit reference of the paged cache's operators on the CPU, and error bounds for their outputs."""
import math

import numpy as np
import torch

IO = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
PAGE = {"f32": torch.float16, "f16": torch.float16, "bf16": torch.bfloat16}
HALF = {t: torch.finfo(IO[t]).eps / 2 for t in IO}          # half a step of the output's type
P_HALF = {"f32": 2.0 ** -21, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}  # of the weights in the products


def page_lists(rng, lengths, page, n_pages):
    """Pages for each sequence, in no order."""
    order, at, out = rng.permutation(n_pages), 0, []
    for n in lengths:
        k = -(-n // page)
        out.append(order[at:at + k].astype(np.int32))
        at += k
    assert at <= n_pages
    return out


def rows_of(pages, table, head, n):
    """Rows 0 .. n - 1 of a sequence and KV head from pages [n_pages][kv][page][d]."""
    return pages[torch.from_numpy(np.asarray(table, np.int64)), head].reshape(-1, pages.shape[-1])[:n].double()


def attention(kind, q, keys, values, qpos, d):
    """(out, bound) of query rows q [r][d] at positions qpos [r] over keys and values [n][d], in 64 bits.

    The bound: the output's own rounding, half a step of P per weight (the sum of the weights takes them
    unrounded), and twice (numerator and sum) a weight's relative error from its score: fp32 sums of d products (d + 8
    roundings of at most the sum of magnitudes; "f32" adds q's split at 2^-22), exp2 and the sums over keys (n
    roundings of fp32, 2^-24 each)."""
    q, n = q.double(), keys.shape[0]
    if n == 0:
        return torch.zeros_like(q), torch.zeros_like(q)
    seen = torch.arange(n)[None, :] <= qpos[:, None]
    s = (q @ keys.t() / math.sqrt(d)).masked_fill(~seen, -math.inf)
    p = torch.softmax(s, -1)
    out = p @ values
    mass = p @ values.abs()
    size = (q.abs() @ keys.abs().t() / math.sqrt(d)).masked_fill(~seen, 0).amax(-1, keepdim=True)
    delta = (d + 8) * 2.0 ** -24 * size + (2.0 ** -22 * size if kind == "f32" else 0) + (n + 16) * 2.0 ** -24
    bound = HALF[kind] * out.abs() + (P_HALF[kind] + 2 * delta) * 1.01 * mass + n * 2.0 ** -36 * values.abs().amax()
    return out, bound


def attend(kind, q, k_pages, v_pages, n_new, lengths, tables, heads, kv, d):
    """(out, bound) [n][heads * d] of a whole batch."""
    g = heads // kv
    n = sum(n_new)
    out, bound = torch.zeros(n, kv, g, d, dtype=torch.float64), torch.zeros(n, kv, g, d, dtype=torch.float64)
    qv, row = q[:n].double().reshape(n, kv, g, d), 0
    for m, length, table in zip(n_new, lengths, tables):
        if m == 0:
            continue
        pos = torch.arange(length - m, length)
        for h in range(kv):
            keys, values = rows_of(k_pages, table, h, length), rows_of(v_pages, table, h, length)
            o, b = attention(kind, qv[row:row + m, h].reshape(m * g, d), keys, values, pos.repeat_interleave(g), d)
            out[row:row + m, h], bound[row:row + m, h] = o.view(m, g, d), b.view(m, g, d)
        row += m
    return out.view(n, heads * d), bound.view(n, heads * d)


def pairs(style, rot):
    """(e0, e1) of each rotation pair of a head of rot elements, the angle's index being the pair's."""
    half, out = rot // 2, []
    for p in range(half):
        if style == 0:
            out.append((p, p + half))
        elif style == 1 and (p | 3) < half:
            e = (p >> 2) * 8 + (p & 3)
            out.append((e, e + 4))
        else:
            out.append((2 * p, 2 * p + 1))
    return torch.tensor(out, dtype=torch.long).reshape(-1, 2)


def turned(x, heads, d, norm, cos, sin, pos, style, rot):
    """Rows normed and rotated, [n][heads][d] in 64 bits, and a bound for fp32 arithmetic on the way: the norm
    (d + 6 roundings), then three roundings of each product's size."""
    x = x.double().reshape(x.shape[0], heads, d)
    grow = 0.0
    if norm is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * torch.as_tensor(norm).double()
        grow = (d + 6) * 2.0 ** -24
    y, mag = x.clone(), x.abs().clone()
    if rot:
        e = pairs(style, rot)
        c, s = cos.double()[pos][:, None, :], sin.double()[pos][:, None, :]
        a, b = x[..., e[:, 0]], x[..., e[:, 1]]
        y[..., e[:, 0]], y[..., e[:, 1]] = a * c - b * s, a * s + b * c
        mag[..., e[:, 0]] = (a * c).abs() + (b * s).abs()
        mag[..., e[:, 1]] = (a * s).abs() + (b * c).abs()
    return y, mag * (grow + 4 * 2.0 ** -24) * 1.01


def exponent(x):
    """floor(log2(x)) within [-24, 24]; 24 for infinities."""
    x = np.asarray(x, np.float64)
    with np.errstate(divide="ignore"):
        e = np.where(x == 0, -24, np.floor(np.log2(np.where(np.isinf(x), 2.0 ** 30, np.maximum(x, 1e-300)))))
    return np.clip(e, -24, 24)


def bounds(rows):
    """(int8 [2][d], scale) of a page's rows [n][d] in use."""
    x = np.asarray(rows, np.float64)
    lo = np.where(np.isnan(x), np.inf, x).min(0)
    hi = np.where(np.isnan(x), -np.inf, x).max(0)
    e = float(exponent(np.maximum(np.abs(lo), np.abs(hi)).max()))
    up = 2.0 ** (6 - e)
    return np.stack([np.clip(np.floor(lo * up), -127, 127), np.clip(np.ceil(hi * up), -127, 127)]).astype(np.int8), 2.0 ** (e - 6)


def choose(q, own, lo_hi, scales, select, first, last):
    """Pages of one query token and KV head: q [g][d], bounds [pages][2][d] and scales [pages] of the sequence's pages."""
    q = q.double().numpy()
    n = own + 1
    if n <= select:
        return list(range(n)) + [-1] * (select - n)
    e = exponent(np.abs(q).max(-1))[:, None]
    qi = np.clip(np.rint(q * 2.0 ** (6 - e)), -127, 127) * 2.0 ** (e - 6)
    b = lo_hi[:n].astype(np.float64)
    score = np.maximum(qi[:, None] * b[None, :, 0], qi[:, None] * b[None, :, 1]).sum(-1).max(0) * scales[:n].astype(np.float64)
    forced = [p for p in range(n) if p < first or p >= n - last]
    rest = sorted((p for p in range(n) if first <= p < n - last), key=lambda p: (-score[p], p))
    return sorted(forced + rest[:select - len(forced)])
