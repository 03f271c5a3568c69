"""Attention over a paged KV cache, as cases that can be timed and checked: the operators of a
server that answers many requests at once.

  append   The new tokens of every sequence of a batch into the pages: per-head RMS norm of q and k
           where the model has one, rotation of the first `rot` elements of a head, K and V rounded
           to the pages' type, and q normed and rotated for the attention. With "bounds", each
           touched page's summary (below) as well.
  attend   Causal attention of the batch's new tokens over their sequences' pages: single tokens,
           chunks of a prompt, or both in one batch.
  sparse   The same with a page budget: every query token and KV head picks the pages whose bound
           promises the largest logits, and attends to those only.

Layouts: pages [n_pages][kv_heads][page][head_dim] for K and for V; tokens [n][heads * head_dim],
the sequences' tokens one after the other. Types: "f32" is fp32 tokens over fp16 pages, "f16" and
"bf16" are one type throughout.

A page's summary, per KV head: with lo and hi the least and largest key of each dim over the page's
rows that are in use (NaN left out), and e = floor(log2(max(|lo|, |hi|))) over the dims, within
[-24, 24], the whole numbers floor(lo 2^(6-e)) and ceil(hi 2^(6-e)) within [-127, 127], and the
scale 2^(e-6). A query head's row is rounded likewise: rint(q 2^(6-e)). A page's score for a
query token and KV head is the largest over the group's query heads of
sum_d max(q_d lo_d, q_d hi_d) times both scales. All of that is exact in fp32, so the choice does
not depend on any order of summation. Chosen are the first `first` pages, the `last` pages that end with
the token's own, and then those of the largest scores, the lower page where scores are equal, `select`
in all; listed in ascending order, -1 behind the last.
"""
import math

import torch

own = False

TYPES = {"f32": (torch.float32, torch.float16), "f16": (torch.float16, torch.float16),
         "bf16": (torch.bfloat16, torch.bfloat16)}
PAIRINGS = {"half": 0, "interleaved": 2}
EPS = 1e-6

# query heads, KV heads, head size: the shapes that the benchmark and the tests run, and head sizes
# outside 64 and 128
SHAPES = [(14, 2, 64), (32, 4, 64), (16, 8, 128), (32, 8, 128), (16, 4, 96), (8, 2, 256), (8, 8, 128)]


def _case(name, op, kind, shape, page, seqs, hist, chunks=0, chunk=(1, 1), rope="half", rot=0, norm=False, bounds=False,
          select=0, first=0, last=0):
    heads, kv_heads, head_dim = shape
    c = {"op": op, "type": kind, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "page": page, "seqs": seqs,
         "hist_lo": hist[0], "hist_hi": hist[1], "chunks": chunks, "chunk_lo": chunk[0], "chunk_hi": chunk[1],
         "rope": rope, "rot": rot, "norm": norm, "bounds": bounds, "select": select, "first": first, "last": last}
    return dict(c, name=name) if name else c


def listed():
    q25, tiny, q317, q38 = (14, 2, 64), (32, 4, 64), (16, 8, 128), (32, 8, 128)
    return [
        # one user's token on a small model: nothing but latency
        _case("append_token", "append", "f32", q25, 16, 1, (700, 700), rot=64),
        # a step of a busy server: one token of each of 48 requests, with QK norm
        _case("append_48_tokens", "append", "bf16", q38, 64, 48, (20, 3000), rot=128, norm=True),
        # four prompts that come in together, half of each head rotated, page summaries kept
        _case("append_prompts_bounds", "append", "f16", tiny, 32, 4, (0, 300), 4, (500, 1100), rope="interleaved", rot=32,
              bounds=True),
        # long prompts in fp32, as the projections of this library write them
        _case("append_prompts", "append", "f32", q38, 16, 6, (0, 500), 6, (300, 1500), rot=128, norm=True),
        # one user's token on a small model
        _case("attend_token_700", "attend", "f32", q25, 16, 1, (700, 700)),
        # a step of a busy server: contexts from short to long
        _case("attend_48_tokens", "attend", "bf16", q38, 64, 48, (200, 30000)),
        # one token behind the longest context
        _case("attend_token_131k", "attend", "f16", q38, 128, 1, (131071, 131071)),
        # a chunk of a long prompt behind the chunks before it
        _case("attend_chunk_2048", "attend", "bf16", q38, 64, 1, (6000, 6000), 1, (2048, 2048)),
        # chunks of three prompts beside the tokens of nine other requests
        _case("attend_mixed", "attend", "f32", tiny, 16, 12, (10, 4000), 3, (150, 500)),
        # one user's token with a page budget
        _case("sparse_token_9000", "sparse", "f32", q317, 16, 1, (9000, 9000), select=24, first=1, last=2),
        # a step of a busy server over long documents, a sixteenth of the pages or less each
        _case("sparse_32_tokens", "sparse", "bf16", q38, 64, 32, (8000, 60000), select=32, first=1, last=2),
        # a chunk of a prompt, each token with its own pages
        _case("sparse_chunk_300", "sparse", "f16", q38, 32, 1, (16000, 16000), 1, (300, 300), select=48, first=1, last=4),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


# what the largest listed case of an operator costs, in bytes and in operations
MOST = {"append": (1.5e8, 1e12), "attend": (1.2e9, 2.3e11), "sparse": (1.2e9, 2.5e10)}


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "sparse"])
    kind, shape, page = rng.choice(list(TYPES)), rng.choice(SHAPES), rng.choice([16, 32, 64, 128])
    seqs = 1 if rng.random() < 0.25 else _log_int(rng, 2, 64)
    a, b = sorted((_log_int(rng, 1, 131071), _log_int(rng, 1, 131071)))
    if op == "append":
        a, b = min(a, 4000), min(b, 4000)
    chunks = rng.choice([0, 0, 1, seqs, (seqs + 2) // 3])
    c, d = sorted((_log_int(rng, 2, 2048), _log_int(rng, 2, 2048)))
    more = {}
    if op == "append":
        more = {"rope": rng.choice(list(PAIRINGS)), "rot": rng.choice([shape[2], shape[2], shape[2] // 2, shape[2] // 4]),
                "norm": rng.random() < 0.5, "bounds": rng.random() < 0.3}
    if op == "sparse":
        c, d = min(c, 400), min(d, 400)
        more = {"select": rng.choice([4, 9, 16, 24, 32, 64]), "first": rng.choice([0, 1, 2]), "last": rng.choice([1, 1, 2])}
    while True:
        case = _case("", op, kind, shape, page, seqs, (a, b), chunks, (c, d) if chunks else (1, 1), **more)
        w, rows = work(case), max(n for n, _ in lengths(case))
        longest = max(length for _, length in lengths(case))
        # the padded operands of the plain form stay within some 20 GB as well
        padded = 4 * (0 if op == "append" else seqs * longest * shape[1] * shape[2] * 3 + seqs * rows * shape[0] * longest * 2
                      if op == "attend" else sum(n for n, _ in lengths(case)) * shape[1] * more["select"] * page * shape[2] * 3)
        if w["bytes"] <= MOST[op][0] and w["flops"] <= MOST[op][1] and padded < 2e10:
            return case
        a, b, c, d = max(1, a * 2 // 3), max(1, b * 3 // 4), max(2, c * 3 // 4), max(2, d * 3 // 4)
        if padded >= 2e10 and b < 20000:
            seqs, chunks = max(1, seqs * 3 // 4), min(chunks, max(1, seqs * 3 // 4))


def lengths(case):
    """(new tokens, length with them) of each sequence: spread over the case's ranges, in no order."""
    out = []
    for i in range(case["seqs"]):
        f, h = (0.5 + 0.6180339887 * i) % 1.0, (0.5 + 0.7548776662 * i) % 1.0
        lo, hi = case["hist_lo"] + 1, case["hist_hi"] + 1
        hist = int(round(lo * (hi / lo) ** f)) - 1
        new = int(round(case["chunk_lo"] * (case["chunk_hi"] / case["chunk_lo"]) ** h)) if i < case["chunks"] else 1
        out.append((new, hist + new))
    return out


def _seen(case):
    """The keys that the new tokens see, summed over the tokens, and the keys of all sequences."""
    pairs = sum(n * (length - n) + n * (n + 1) // 2 for n, length in lengths(case))
    return pairs, sum(length for _, length in lengths(case))


def _sparse_keys(case):
    """The same for the chosen pages: keys seen, and rows of the bounds that a token's choice has to look at."""
    keys, pages = 0, 0
    for n, length in lengths(case):
        for pos in {length - n, length - 1}:
            vis = pos // case["page"] + 1
            part = n / 2 if n > 1 else 1
            keys += part * ((min(vis, case["select"]) - 1) * case["page"] + pos % case["page"] + 1)
        pages += (length + case["page"] - 1) // case["page"]
    return int(keys), pages


def work(case):
    new = sum(n for n, _ in lengths(case))
    size = 4 if case["type"] == "f32" else 2
    h, kv, d = case["heads"], case["kv_heads"], case["head_dim"]
    if case["op"] == "append":
        moved = new * (2 * h * d * size + 2 * kv * d * (size + 2))
        return {"bytes": moved, "flops": new * (h + kv) * d * 6}
    if case["op"] == "attend":
        pairs, keys = _seen(case)
        return {"bytes": keys * kv * d * 4 + 2 * new * h * d * size, "flops": 4 * pairs * h * d}
    keys, pages = _sparse_keys(case)
    # tokens of one sequence may choose the same pages, so of a chunk's pages only the sequence's are counted
    least = min(keys * 4, _seen(case)[1] * 4)
    bounds = pages * kv * (2 * d + 4) if any(length > case["select"] * case["page"] for _, length in lengths(case)) else 0
    return {"bytes": least * kv * d + bounds + 2 * new * h * d * size + new * kv * case["select"] * 4,
            "flops": 4 * keys * h * d}


# ---- inputs ----

class _State:
    pass


def _inputs(case, seed):
    """The tensors of a case, from the seed alone."""
    s = _State()
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 7919 + 11)
    cpu = torch.Generator()
    cpu.manual_seed(seed * 7919 + 13)
    s.io, s.store = TYPES[case["type"]]
    h, kv, d, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    s.lens = lengths(case)
    s.new = sum(n for n, _ in s.lens)
    held = [(length + page - 1) // page for _, length in s.lens]
    s.n_pages = sum(held) + 3
    order = torch.randperm(s.n_pages, generator=cpu).tolist()
    s.tables, at = [], 0
    for n in held:
        s.tables.append(order[at:at + n])
        at += n
    s.k_pages = torch.randn((s.n_pages, kv, page, d), generator=g, device="cuda", dtype=s.store)
    s.v_pages = torch.randn((s.n_pages, kv, page, d), generator=g, device="cuda", dtype=s.store)
    s.q = torch.randn((s.new, h * d), generator=g, device="cuda", dtype=s.io)
    s.positions = [length - n + i for n, length in s.lens for i in range(n)]
    if case["op"] == "append":
        s.k = torch.randn((s.new, kv * d), generator=g, device="cuda", dtype=s.io)
        s.v = torch.randn((s.new, kv * d), generator=g, device="cuda", dtype=s.io)
        s.q_norm = 1.0 + 0.1 * torch.randn(d, generator=cpu) if case["norm"] else None
        s.k_norm = 1.0 + 0.1 * torch.randn(d, generator=cpu) if case["norm"] else None
        s.max_pos = max(length for _, length in s.lens)
        angle = torch.arange(s.max_pos, dtype=torch.float64)[:, None] / 1e6 ** (
            torch.arange(0, case["rot"], 2, dtype=torch.float64)[None, :] / case["rot"])
        s.cos, s.sin = torch.cos(angle).float(), torch.sin(angle).float()
    return s


def _exponent(x):
    """floor(log2(x)) within [-24, 24]."""
    return torch.clamp(torch.frexp(x)[1] - 1, -24, 24)


def _power(e):
    """2^e in fp32."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _summaries(k, used):
    """Whole numbers lo and hi [n][kv][2][d] and the scales [n][kv] of pages k [n][kv][page][d], of which the first
    `used` rows [n] are in use."""
    x = k.float()
    left_out = torch.isnan(x) | (torch.arange(k.shape[2], device=k.device)[None, None, :, None] >= used[:, None, None, None])
    lo = torch.where(left_out, math.inf, x).amin(2)
    hi = torch.where(left_out, -math.inf, x).amax(2)
    e = _exponent(torch.maximum(lo.abs(), hi.abs()).amax(-1))
    up = _power(6 - e)[..., None]
    both = torch.stack((torch.floor(lo * up), torch.ceil(hi * up)), 2)
    return torch.clamp(both, -127, 127).to(torch.int8), _power(e - 6)


def prepare(case, seed):
    s = _inputs(case, seed)
    s.case = case
    dev, page = "cuda", case["page"]
    if case["op"] == "sparse" or case["bounds"]:
        used = torch.full((s.n_pages,), page, device=dev)
        s.bounds, s.scales = _summaries(s.k_pages, used)
    if own:
        from picolm_qwen_amd import PagedAttention

        rope = {}
        if case["op"] == "append":
            rope = {"rope_style": PAIRINGS[case["rope"]], "rot_dim": case["rot"], "rope_cos": s.cos, "rope_sin": s.sin}
        s.att = PagedAttention(1, s.n_pages, page, case["heads"], case["kv_heads"], case["head_dim"], dtype=case["type"],
                               key_pages=s.k_pages, val_pages=s.v_pages, key_bounds=getattr(s, "bounds", None),
                               key_scales=getattr(s, "scales", None), **rope)
        if case["norm"]:
            s.att.set_qk_norm(0, s.q_norm, s.k_norm)
        s.batch = s.att.batch(case["seqs"], s.new)
        s.batch.set([n for n, _ in s.lens], [length for _, length in s.lens], s.tables)
        return s
    # the same plan as index tensors
    longest = max(len(t) for t in s.tables)
    s.table = torch.tensor([t + [0] * (longest - len(t)) for t in s.tables], device=dev)
    s.pos = torch.tensor(s.positions, device=dev)
    s.seq = torch.tensor([i for i, (n, _) in enumerate(s.lens) for _ in range(n)], device=dev)
    s.length = torch.tensor([length for _, length in s.lens], device=dev)
    s.count = torch.tensor([n for n, _ in s.lens], device=dev)
    s.nth = s.pos - (s.length - s.count)[s.seq]  # each token's place among its sequence's new ones
    if case["op"] == "append":
        s.cos, s.sin = s.cos.to(dev), s.sin.to(dev)
        if case["norm"]:
            s.q_norm, s.k_norm = s.q_norm.to(dev), s.k_norm.to(dev)
        if case["bounds"]:
            touched = [(t[j], min(page, length - j * page)) for t, (n, length) in zip(s.tables, s.lens)
                       for j in range((length - n) // page, (length + page - 1) // page)]
            s.touched = torch.tensor([p for p, _ in touched], device=dev)
            s.used = torch.tensor([u for _, u in touched], device=dev)
    return s


# ---- the plain forms ----

def _turned(x, w, s, heads):
    """Rows x [n][heads * d], normed with w where given and rotated: fp32 [n][heads][d]."""
    case = s.case
    rot, half = case["rot"], case["rot"] // 2
    x = x.float().view(x.shape[0], heads, case["head_dim"])
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w
    c, n = s.cos[s.pos][:, None, :], s.sin[s.pos][:, None, :]
    y = x.clone()
    if case["rope"] == "half":
        a, b = x[..., :half], x[..., half:rot]
        y[..., :half], y[..., half:rot] = a * c - b * n, a * n + b * c
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y[..., 0:rot:2], y[..., 1:rot:2] = a * c - b * n, a * n + b * c
    return y


def _plain_append(s):
    case = s.case
    kv, page = case["kv_heads"], case["page"]
    q = _turned(s.q, s.q_norm, s, case["heads"]).to(s.io).view(s.new, -1)
    k = _turned(s.k, s.k_norm, s, kv).to(s.store)
    where, slot = s.table[s.seq, s.pos // page], s.pos % page
    s.k_pages[where, :, slot] = k
    s.v_pages[where, :, slot] = s.v.view(s.new, kv, -1).to(s.store)
    if case["bounds"]:
        s.bounds[s.touched], s.scales[s.touched] = _summaries(s.k_pages[s.touched], s.used)
    return q


def _soft(scores, seen):
    """Weights of the seen keys, and zero for the others."""
    scores = torch.where(seen, scores, -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    return p / p.sum(-1, keepdim=True)


def _plain_attend(s):
    case = s.case
    h, kv, d, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    n, rows, keys = len(s.lens), max(x for x, _ in s.lens), s.table.shape[1] * page
    q = torch.zeros((n, rows, kv, h // kv, d), device="cuda")
    q[s.seq, s.nth] = s.q.float().view(s.new, kv, h // kv, d)
    q = q.permute(0, 2, 1, 3, 4).reshape(n, kv, rows * (h // kv), d)
    k = s.k_pages[s.table].permute(0, 2, 1, 3, 4).reshape(n, kv, keys, d).float()
    v = s.v_pages[s.table].permute(0, 2, 1, 3, 4).reshape(n, kv, keys, d).float()
    at = torch.arange(keys, device="cuda")
    last = (s.length - s.count)[:, None] + torch.arange(rows, device="cuda")  # rows past the last token see keys that no one reads
    seen = at <= last.repeat_interleave(h // kv, 1)[:, None, :, None]
    o = torch.matmul(_soft(torch.matmul(q, k.transpose(-1, -2)) / math.sqrt(d), seen), v)
    o = o.view(n, kv, rows, h // kv, d).permute(0, 2, 1, 3, 4)
    return o[s.seq, s.nth].reshape(s.new, h * d).to(s.io)


def _plain_sparse(s):
    case = s.case
    h, kv, d, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    q = s.q.float().view(s.new, kv, h // kv, d)
    # the scores of all pages of the token's sequence: [new][kv][pages]
    e = _exponent(q.abs().amax(-1))
    qi = torch.clamp(torch.round(q * _power(6 - e)[..., None]), -127, 127)
    signed = torch.cat((torch.clamp(qi, max=0), torch.clamp(qi, min=0)), -1)
    pages = s.table[s.seq]
    b = s.bounds[pages].permute(0, 2, 3, 4, 1).reshape(s.new, kv, 2 * d, -1).float()
    best = (torch.matmul(signed, b) * _power(e - 6)[..., None]).amax(2) * s.scales[pages].permute(0, 2, 1)
    at, mine = torch.arange(pages.shape[1], device="cuda"), (s.pos // page)[:, None]
    best = torch.where(((at < case["first"]) | (at > mine - case["last"]))[:, None, :], math.inf, best)
    best = torch.where((at > mine)[:, None, :], -math.inf, best)
    ranked = torch.sort(best, stable=True, dim=-1, descending=True)[1][..., :case["select"]]
    ranked = torch.sort(torch.where(ranked > mine[..., None], pages.shape[1], ranked), -1)[0]
    chosen = torch.full((s.new, kv, case["select"]), -1, device="cuda", dtype=torch.int32)
    chosen[..., :ranked.shape[-1]] = torch.where(ranked == pages.shape[1], -1, ranked)
    # attention over the chosen pages
    real = torch.clamp(chosen, min=0).long()
    physical = torch.gather(pages[:, None, :].expand(-1, kv, -1), 2, real)
    head = torch.arange(kv, device="cuda")[None, :, None]
    k = s.k_pages[physical, head].reshape(s.new, kv, -1, d).float()
    v = s.v_pages[physical, head].reshape(s.new, kv, -1, d).float()
    key = real[..., None] * page + torch.arange(page, device="cuda")
    seen = ((key <= s.pos[:, None, None, None]) & (chosen >= 0)[..., None]).view(s.new, kv, 1, -1)
    o = torch.matmul(_soft(torch.matmul(q, k.transpose(-1, -2)) / math.sqrt(d), seen), v)
    return o.reshape(s.new, h * d).to(s.io), chosen


def run(s):
    case = s.case
    if case["op"] == "append":
        q = s.att.append(0, s.batch, s.q, s.k, s.v) if own else _plain_append(s)
        if case["bounds"]:  # as the values that the whole numbers stand for
            return q, s.k_pages, s.v_pages, (s.bounds * s.scales[..., None, None]).to(s.store)
        return q, s.k_pages, s.v_pages
    if case["op"] == "attend":
        return s.att.attend(0, s.batch, s.q) if own else _plain_attend(s)
    if own:
        return s.att.attend_sparse(0, s.batch, s.q, case["select"], case["first"], case["last"])
    return _plain_sparse(s)


# ---- the definitions in 64 bits ----

def _exact_turned(x, w, s, case, heads):
    """Norm and rotation as complex numbers."""
    rot, d = case["rot"], case["head_dim"]
    x = x.double().view(-1, heads, d)
    if w is not None:
        x = x * torch.rsqrt(x.square().sum(-1, keepdim=True) / d + EPS) * w.double().to(x.device)
    at = torch.tensor(s.positions)
    z = torch.complex(s.cos.double()[at], s.sin.double()[at]).to(x.device)[:, None, :]
    if case["rope"] == "half":
        pairs = torch.complex(x[..., :rot // 2], x[..., rot // 2:rot]) * z
        turned = torch.cat((pairs.real, pairs.imag), -1)
    else:
        turned = torch.view_as_real(torch.view_as_complex(x[..., :rot].reshape(*x.shape[:-1], rot // 2, 2).contiguous()) * z).flatten(-2)
    return torch.cat((turned, x[..., rot:]), -1)


def _exact_append(case, s):
    kv, page = case["kv_heads"], case["page"]
    q = _exact_turned(s.q, s.q_norm, s, case, case["heads"]).flatten(1)
    k, v = _exact_turned(s.k, s.k_norm, s, case, kv), s.v.double().view(s.new, kv, -1)
    kp, vp = s.k_pages.double(), s.v_pages.double()
    row = 0
    for (n, length), table in zip(s.lens, s.tables):
        for j in range((length - n) // page, (length + page - 1) // page):
            a, b = max(j * page, length - n), min((j + 1) * page, length)
            r = row + a - (length - n)
            kp[table[j], :, a - j * page:b - j * page] = k[r:r + b - a].transpose(0, 1)
            vp[table[j], :, a - j * page:b - j * page] = v[r:r + b - a].transpose(0, 1)
        row += n
    # a summary is made from the rows as the pages hold them, so it has no value apart from their rounding
    return (q, kp, vp, None) if case["bounds"] else (q, kp, vp)


def _exact_rows(s, which, table, head, keys):
    pages = (s.k_pages if which == 0 else s.v_pages)[torch.tensor(table, device="cuda"), head]
    return pages.reshape(-1, pages.shape[-1])[:keys].double()


def _exact_attend(case, s):
    h, kv, d = case["heads"], case["kv_heads"], case["head_dim"]
    g = h // kv
    q = s.q.double().view(s.new, kv, g, d)
    out = torch.zeros((s.new, kv, g, d), dtype=torch.float64, device="cuda")
    row = 0
    for (n, length), table in zip(s.lens, s.tables):
        hidden = torch.triu(torch.ones((n, length), dtype=torch.bool, device="cuda"), length - n + 1)
        for head in range(kv):
            k, v = (_exact_rows(s, w, table, head, length) for w in (0, 1))
            for i in range(g):
                logits = (q[row:row + n, head, i] @ k.t().contiguous() * d ** -0.5).masked_fill_(hidden, -math.inf)
                out[row:row + n, head, i] = torch.softmax(logits, -1) @ v
        row += n
    return out.view(s.new, h * d)


def _exact_sparse(case, s):
    h, kv, d, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    g, budget = h // kv, case["select"]
    bounds, scales = _summaries(s.k_pages, torch.full((s.n_pages,), page, device="cuda"))
    q = s.q.double().view(s.new, kv, g, d)
    step = torch.exp2(torch.clamp(torch.floor(torch.log2(q.abs().amax(-1, keepdim=True))), -24, 24) - 6)
    coarse = torch.clamp(torch.round(q / step), -127, 127) * step
    out = torch.zeros((s.new, kv, g, d), dtype=torch.float64, device="cuda")
    chosen = torch.full((s.new, kv, budget), -1, dtype=torch.int32)
    row = 0
    for (n, length), table in zip(s.lens, s.tables):
        t = torch.tensor(table, device="cuda")
        real = bounds[t].double() * scales[t].double()[..., None, None]
        for head in range(kv):
            k, v = (_exact_rows(s, w, table, head, len(table) * page) for w in (0, 1))
            for i in range(row, row + n):
                pos = s.positions[i]
                mine = pos // page
                worth = torch.maximum(coarse[i, head, :, None] * real[None, :, head, 0],
                                      coarse[i, head, :, None] * real[None, :, head, 1]).sum(-1).amax(0).tolist()
                must = [p for p in range(mine + 1) if p < case["first"] or p > mine - case["last"]]
                rest = sorted((p for p in range(mine + 1) if p not in set(must)), key=lambda p: (-worth[p], p))
                pages = sorted((must + rest)[:budget])
                chosen[i, head, :len(pages)] = torch.tensor(pages, dtype=torch.int32)
                keys = torch.tensor([p * page + r for p in pages for r in range(page) if p * page + r <= pos], device="cuda")
                out[i, head] = torch.softmax(q[i, head] @ k[keys].t().contiguous() / math.sqrt(d), -1) @ v[keys]
        row += n
    return out.view(s.new, h * d), chosen.to("cuda")


def exact(case, seed):
    if case["op"] == "sparse" and sum(n * (length // case["page"] + 50) for n, length in lengths(case)) * case["kv_heads"] > 2_000_000:
        return None
    s = _inputs(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "sparse": _exact_sparse}[case["op"]](case, s)
