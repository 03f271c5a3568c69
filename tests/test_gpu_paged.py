"""The paged cache's operators on the GPU against 64-bit references (tests/paged_ref.py): append, attention and
attention with a page budget over batches of single tokens and chunks, all types, page and head sizes."""
import gc

import numpy as np
import pytest

import oracle as O
import paged_ref as R
from conftest import cpu_threads

torch = pytest.importorskip("torch")
from picolm_qwen_amd import PagedAttention, PicoAttention, PQAError, rope_table  # noqa: E402
from picolm_qwen_amd.hipgraph import Graph  # noqa: E402

pytestmark = pytest.mark.gpu

# (heads, KV heads, head size)
SHAPES = [(14, 2, 64), (16, 4, 96), (32, 8, 128), (5, 1, 160), (6, 6, 192), (8, 2, 256), (34, 2, 64), (17, 1, 128)]
# (new, length) of each sequence: single tokens at tile and page borders, empty ones, chunks, long
BATCHES = {
    "tokens": [(1, 1), (1, 2), (1, 15), (1, 16), (1, 17), (1, 31), (1, 32), (1, 33), (1, 64), (1, 65), (0, 40), (1, 129), (1, 700)],
    "one": [(1, 1)],
    "long": [(1, 5000)],
    "chunks": [(70, 70), (1, 300), (33, 500), (0, 0), (129, 130), (2, 2), (3, 1200)],
    "chunk": [(257, 900)],
    "turns": [(5, 2100), (20, 2100)],
}


class Cache:
    """A handle over random pages, and the same pages on the CPU. Rows that no sequence uses are NaN."""

    def __init__(self, kind, shape, page, seqs, seed=0, spare=2, layers=1, layer=0, stale=float("nan"), **more):
        self.kind, (self.heads, self.kv, self.d), self.page = kind, shape, page
        self.seqs, self.n_new, self.lengths = seqs, [n for n, _ in seqs], [length for _, length in seqs]
        self.n = sum(self.n_new)
        rng = np.random.default_rng(seed)
        self.n_pages = sum(-(-length // page) for length in self.lengths) + spare
        self.tables = R.page_lists(rng, self.lengths, page, self.n_pages)
        g = torch.Generator().manual_seed(seed)
        full = (layers, self.n_pages, self.kv, page, self.d)
        self.k = torch.full(full, stale, dtype=R.PAGE[kind])
        self.v = torch.full(full, stale, dtype=R.PAGE[kind])
        self.layer = layer
        for length, t in zip(self.lengths, self.tables):
            for j, p in enumerate(t):
                used = min(page, length - j * page)
                for x in (self.k, self.v):
                    x[layer, p, :, :used] = torch.randn(self.kv, used, self.d, generator=g).to(R.PAGE[kind])
        self.q = torch.randn(self.n, self.heads * self.d, generator=g).to(R.IO[kind])
        self.pos = torch.tensor([length - n + i for n, length in seqs for i in range(n)], dtype=torch.long)
        self.dk, self.dv = self.k.cuda(), self.v.cuda()
        self.att = PagedAttention(layers, self.n_pages, page, *shape, dtype=kind, key_pages=self.dk, val_pages=self.dv, **more)
        self.batch = self.att.batch(len(seqs) + 1, max(self.n, 1))
        self.batch.set(self.n_new, self.lengths, self.tables)

    def want(self, q=None):
        return R.attend(self.kind, self.q if q is None else q, self.k[self.layer], self.v[self.layer], self.n_new, self.lengths,
                        self.tables, self.heads, self.kv, self.d)


def near(got, want, bound, what=""):
    got = got.double().cpu()
    assert torch.isfinite(got).all(), f"{what}: not finite"
    err = (got - want).abs()
    bad = err > bound
    if bad.any():
        i = int((err / bound.clamp_min(1e-300)).argmax())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} outside; worst at {i}: got {got.flatten()[i]:.8g} "
                             f"want {want.flatten()[i]:.8g} bound {bound.flatten()[i]:.3g}")


# ---- attention ----

@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("name", ["tokens", "chunks"])
def test_attend(kind, shape, name):
    c = Cache(kind, shape, 16 if shape[2] != 96 else 64, BATCHES[name], seed=3)
    out = c.att.attend(0, c.batch, c.q.cuda())
    near(out, *c.want(), what=f"{kind} {shape} {name}")


@pytest.mark.parametrize("kind,shape,page,name", [
    ("f32", (32, 8, 128), 16, "one"), ("bf16", (32, 4, 64), 256, "one"), ("f16", (4, 4, 128), 32, "tokens"),
    ("f16", (32, 8, 128), 128, "long"), ("f32", (14, 2, 64), 32, "long"), ("bf16", (2, 1, 256), 64, "long"),
    ("bf16", (32, 8, 128), 64, "chunk"), ("f32", (16, 8, 128), 16, "chunk"), ("f16", (8, 1, 64), 256, "chunk"),
    ("f32", (8, 2, 256), 32, "turns"), ("bf16", (8, 2, 128), 32, "turns"), ("f16", (2, 2, 64), 16, "turns")],
    ids=lambda x: "x".join(map(str, x)) if isinstance(x, tuple) else str(x))
def test_attend_pages_and_lengths(kind, shape, page, name):
    c = Cache(kind, shape, page, BATCHES[name], seed=5)
    near(c.att.attend(0, c.batch, c.q.cuda()), *c.want(), what=f"{kind} {shape} {page} {name}")


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_errors_stay_at_the_types_level(kind):
    # relative 2-norm: independent roundings of half a step, over sqrt(3) each; fp32-level for "f32", whose
    # worst roundings (2^-22 of q, d sums of 2^-24) leave 1e-6 of a value
    c = Cache(kind, (32, 8, 128), 32, [(1, 3000), (200, 1000), (7, 90)], seed=11)
    out, (want, _) = c.att.attend(0, c.batch, c.q.cuda()).double().cpu(), c.want()
    rel = float((out - want).norm() / want.norm())
    assert rel <= {"f32": 3e-6, "f16": 1.5 * 2.0 ** -11, "bf16": 1.5 * 2.0 ** -8}[kind], rel


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_strides_padding_and_in_place(kind):
    # q as the first part of wider rows at an odd element offset, more rows than tokens, out in place
    c = Cache(kind, (14, 2, 64), 16, BATCHES["chunks"], seed=7)
    dim, rows = 14 * 64, c.n + 3
    wide = torch.full((rows, dim + 131), 7.0, dtype=R.IO[kind], device="cuda")
    q = wide[:, 1:1 + dim]
    q[:c.n] = c.q.cuda()
    want = c.want()
    out = torch.full((rows, dim), 5.0, dtype=R.IO[kind], device="cuda")
    assert c.att.attend(0, c.batch, q, out=out) is out
    near(out[:c.n], *want, what="strided q")
    assert bool((out[c.n:] == 5.0).all()), "rows behind the last token were written"
    assert c.att.attend(0, c.batch, q, out=q) is q
    near(q[:c.n], *want, what="in place")
    assert bool((wide[:, 0] == 7).all() and (wide[:, 1 + dim:] == 7).all() and (wide[c.n:] == 7).all())
    fresh = c.att.attend(0, c.batch, torch.cat([c.q.cuda(), torch.ones(2, dim, dtype=R.IO[kind], device="cuda")]))
    near(fresh[:c.n], *want, what="padded")
    assert bool((fresh[c.n:] == 0).all())


def test_shared_pages_and_a_second_layer():
    # two requests behind one prompt of 64 positions, in layer 1 of 3
    c = Cache("bf16", (8, 2, 128), 16, [(1, 70), (0, 64), (30, 94)], seed=9, layers=3, layer=1)
    c.tables[2][:4] = c.tables[0][:4]
    c.batch.set(c.n_new, c.lengths, c.tables)
    near(c.att.attend(1, c.batch, c.q.cuda()), *c.want())


def test_a_long_pool_addresses_past_32_bits():
    # one page holds 512 KB of K: the last ones start past 4 GiB
    kind, shape, page, n = "f16", (16, 8, 128), 256, 9000
    small = Cache(kind, shape, page, [(1, 300), (70, 600)], seed=13)
    k = torch.empty((n, 8, page, 128), dtype=torch.float16, device="cuda")
    v = torch.empty_like(k)
    move = n - small.n_pages
    k[move:], v[move:] = small.dk[0], small.dv[0]
    att = PagedAttention(1, n, page, *shape, dtype=kind, key_pages=k, val_pages=v)
    batch = att.batch(2, small.n, 1000)
    batch.set(small.n_new, small.lengths, [t + move for t in small.tables])
    near(att.attend(0, batch, small.q.cuda()), *small.want())


def test_results_do_not_depend_on_the_order_of_finishing():
    for kind, seqs in (("f32", [(1, 9000), (1, 40)]), ("bf16", [(40, 4000)])):
        c = Cache(kind, (16, 8, 128), 16, seqs, seed=15)
        q = c.q.cuda()
        first = c.att.attend(0, c.batch, q)
        for _ in range(5):
            assert torch.equal(c.att.attend(0, c.batch, q), first)


# ---- values that are not finite: the formula in fp32 over the keys that a row sees ----

def formula(c):
    """The attention of each row over its own keys in fp32 (a weight of zero times infinity is NaN)."""
    g, out = c.heads // c.kv, torch.zeros(c.n, c.kv, c.heads // c.kv, c.d)
    q, row = c.q.float().view(c.n, c.kv, g, c.d), 0
    for m, length, t in zip(c.n_new, c.lengths, c.tables):
        for i in range(m):
            for h in range(c.kv):
                k = R.rows_of(c.k[c.layer], t, h, length - m + i + 1).float()
                v = R.rows_of(c.v[c.layer], t, h, length - m + i + 1).float()
                s = (q[row + i, h] @ k.t()) / c.d ** 0.5
                p = torch.exp(s - s.amax(-1, keepdim=True))
                out[row + i, h] = (p / p.sum(-1, keepdim=True)) @ v
        row += m
    return out.view(c.n, -1)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", [(14, 2, 64), (8, 2, 128), (4, 2, 256)], ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("what,value", [("v", float("inf")), ("v", float("nan")), ("k", float("inf")), ("k", float("-inf")),
                                        ("k", float("nan"))])
def test_infinities_and_nan(kind, shape, what, value):
    # at a position that some rows see and others do not, in one dim of KV head 1 (v) or all of them (k)
    seqs = [(40, 300), (1, 200), (3, 64), (1, 1300)]
    c = Cache(kind, shape, 16, seqs, seed=17)
    for t, at in zip(c.tables, (280, 100, 62, 1200)):
        x = (c.v if what == "v" else c.k)[0, t[at // 16], 1, at % 16]
        if what == "v":
            x[5] = value
        else:
            x[:] = value
    c.dk.copy_(c.k)
    c.dv.copy_(c.v)
    got, want = c.att.attend(0, c.batch, c.q.cuda()).double().cpu(), formula(c).double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.isinf(got), torch.isinf(want))
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf])
    # the finite rows: those that do not see the value, and (k = -inf with q's signs) those whose weight of it is zero
    fine = torch.isfinite(want)
    # of values around 1: fp32 sums over up to 1300 keys and 256 dims on both sides, (1300 + 256) 2^-24 < 1e-4; four half
    # steps of the 16-bit types (the output's and P's, on values up to 2)
    tol = {"f32": 1e-4, "f16": 2.0 ** -9, "bf16": 2.0 ** -6}[kind]
    assert float((got - want)[fine].abs().max()) <= tol * max(1.0, float(want[fine].abs().max()))
    assert fine.any() and (~fine).any()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_large_and_zero_queries(kind):
    c = Cache(kind, (8, 2, 128), 16, [(1, 100), (20, 120)], seed=19)
    q = c.q.clone()
    q[0] = 0
    q[1] *= 3e4
    q[2] *= 1e-30
    q[3, :64] = 1e30 if kind == "f32" else 1e20
    c.q = q
    got, want = c.att.attend(0, c.batch, q.cuda()).double().cpu(), c.want()[0]
    assert torch.isfinite(got).all()
    for row in (0, 2):  # equal weights: the mean of the values seen
        assert float((got[row] - want[row]).abs().max()) <= 2 * R.HALF[kind] * 4 + 1e-5
    for row in (1, 3):  # one weight, but for ties that 64 bits tell apart and fp32 may not
        vals = torch.cat([R.rows_of(c.v[0], c.tables[0 if row == 0 else 1], h, 120) for h in range(2)])
        assert float(got[row].abs().max()) <= float(vals.abs().max()) * (1 + 2 * R.HALF[kind])


# ---- append ----

def append_case(kind, shape, page, seqs, norm, style, rot, bounds, seed=21):
    rng = np.random.default_rng(seed)
    heads, kv, d = shape
    top = max(length for _, length in seqs) + 5
    angle = np.arange(top)[:, None] / 1e4 ** (np.arange(0, rot, 2)[None, :] / max(rot, 1))
    cos, sin = np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)
    more = {"rope_style": style, "rot_dim": rot, "rope_cos": cos, "rope_sin": sin} if rot else {}
    n_pages = sum(-(-length // page) for _, length in seqs) + 2
    if bounds:
        more.update(key_bounds=torch.zeros((n_pages, kv, 2, d), dtype=torch.int8, device="cuda"),
                    key_scales=torch.zeros((n_pages, kv), device="cuda"))
    c = Cache(kind, shape, page, seqs, seed=seed, stale=3.0, **more)
    if norm:
        c.qn, c.kn = (1 + 0.2 * rng.standard_normal((2, d))).astype(np.float32)
        c.att.set_qk_norm(0, c.qn, c.kn)
    else:
        c.qn = c.kn = None
    g = torch.Generator().manual_seed(seed + 1)
    c.nk = torch.randn(c.n, kv * d, generator=g).to(R.IO[kind])
    c.nv = torch.randn(c.n, kv * d, generator=g).to(R.IO[kind])
    c.cos, c.sin, c.style, c.rot = torch.from_numpy(cos), torch.from_numpy(sin), style, rot
    return c


def check_append(c, q_out, before):
    kind, page = c.kind, c.page
    want, err = R.turned(c.q, c.heads, c.d, c.qn, c.cos, c.sin, c.pos, c.style, c.rot)
    # below the smallest normal number the type's step no longer shrinks with the value: half of it is
    # smallest_normal * eps / 2 (fp16: 2^-14 * 2^-11 = 2^-25)
    low = torch.finfo(R.IO[kind]).smallest_normal * R.HALF[kind]
    near(q_out, want.view(c.n, -1), (err + R.HALF[kind] * (want.abs() + err)).view(c.n, -1) + low, "q")
    k, kerr = R.turned(c.nk, c.kv, c.d, c.kn, c.cos, c.sin, c.pos, c.style, c.rot)
    half = torch.finfo(R.PAGE[kind]).eps / 2
    tiny = torch.finfo(R.PAGE[kind]).smallest_normal * half  # half a step of the subnormal values
    got_k, got_v = c.dk.cpu()[c.layer], c.dv.cpu()[c.layer]
    expect_k, expect_v = before[0][c.layer].clone(), before[1][c.layer].clone()
    v = c.nv.to(R.PAGE[kind]).view(c.n, c.kv, c.d)
    row = 0
    for m, length, t in zip(c.n_new, c.lengths, c.tables):
        for i in range(m):
            pos = length - m + i
            p, slot = int(t[pos // page]), pos % page
            near(got_k[p, :, slot], k[row], kerr[row] + half * (k[row].abs() + kerr[row]) + tiny, f"K row {pos}")
            expect_k[p, :, slot] = got_k[p, :, slot]
            expect_v[p, :, slot] = v[row]
            row += 1
    assert torch.equal(got_k.view(torch.int16), expect_k.view(torch.int16)), "other K rows changed"
    if kind == "f32":  # ties of fp32 values go away from zero in the one, to even in the other: half a step either way
        near(got_v, expect_v.double(), half * 2 * expect_v.double().abs() + tiny, "V rows")
    else:
        assert torch.equal(got_v.view(torch.int16), expect_v.view(torch.int16))


def check_bounds(c):
    b, s, rows = c.att.key_bounds.cpu().numpy(), c.att.key_scales.cpu().numpy(), c.dk.cpu()[c.layer]
    for m, length, t in zip(c.n_new, c.lengths, c.tables):
        for j in range((length - m) // c.page, -(-length // c.page) if m else 0):
            for h in range(c.kv):
                want, scale = R.bounds(rows[t[j], h, :min(c.page, length - j * c.page)].double().numpy())
                assert np.array_equal(b[t[j], h], want) and s[t[j], h] == scale, (j, h)


@pytest.mark.parametrize("kind,shape,page,name,norm,style,rot,bounds", [
    ("f32", (14, 2, 64), 16, "tokens", False, 0, 64, False), ("f32", (32, 8, 128), 16, "chunks", True, 0, 128, True),
    ("f16", (16, 4, 96), 32, "chunks", True, 2, 96, True), ("bf16", (8, 2, 256), 64, "chunks", True, 0, 64, True),
    ("bf16", (32, 8, 128), 128, "tokens", True, 1, 128, True), ("f16", (5, 1, 160), 16, "chunk", False, 1, 40, False),
    ("f32", (6, 6, 192), 256, "chunk", True, 2, 10, True), ("bf16", (4, 1, 64), 16, "one", False, 0, 0, True)],
    ids=lambda x: "x".join(map(str, x)) if isinstance(x, tuple) else str(x))
def test_append(kind, shape, page, name, norm, style, rot, bounds):
    c = append_case(kind, shape, page, BATCHES[name], norm, style, rot, bounds)
    before = c.k.clone(), c.v.clone()
    q = c.att.append(0, c.batch, c.q.cuda(), c.nk.cuda(), c.nv.cuda())
    check_append(c, q, before)
    if bounds:
        check_bounds(c)


@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_append_from_packed_rows_in_place(kind):
    # q, k and v as parts of one row each, at offsets and distances that are no multiple of four
    c = append_case(kind, (14, 2, 64), 16, BATCHES["chunks"], True, 0, 32, False)
    before = c.k.clone(), c.v.clone()
    wide = torch.full((c.n + 2, 18 * 64 + 7), 9.0, dtype=R.IO[kind], device="cuda")
    q, k, v = wide[:, 3:3 + 896], wide[:, 3 + 896:3 + 1024], wide[:, 4 + 1024:4 + 1152]
    q[:c.n], k[:c.n], v[:c.n] = c.q.cuda(), c.nk.cuda(), c.nv.cuda()
    assert c.att.append(0, c.batch, q, k, v, q_out=q) is q
    check_append(c, q[:c.n], before)
    assert bool((wide[c.n:] == 9).all()) and bool((wide[:, :3] == 9).all())


def test_rows_have_the_bits_of_the_contiguous_cache():
    # fp32 tokens over fp16 pages, all three pairings, with norm: the oracle's cache rows
    for style in (0, 1, 2):
        seqs, shape, smax = [(1, 37), (50, 90)], (32, 8, 128), 128
        nh, nkv, hd = shape
        cos, sin = O.rope_table(1e6, hd, smax)
        c = Cache("f32", shape, 16, seqs, seed=23, stale=0.0, rope_style=style, rope_cos=cos, rope_sin=sin)
        qn, kn = O.qk_norm_weights(7, 0, hd)
        c.att.set_qk_norm(0, qn, kn)
        at = 0
        q, k, v = O.batch_inputs(7, 1, 0, c.n, nh, nkv, hd)
        c.att.append(0, c.batch, *(torch.from_numpy(x).cuda() for x in (q, k, v)))
        for (m, length), t in zip(seqs, c.tables):
            kc, vc = np.zeros((smax, nkv * hd), np.uint16), np.zeros((smax, nkv * hd), np.uint16)
            O.prefill(O.shape(nh, nkv, hd, smax, style), length - m, q[at:at + m], k[at:at + m], v[at:at + m], qn, kn, cos, sin,
                      kc, vc, n_threads=cpu_threads())
            for got, want in ((c.dk, kc), (c.dv, vc)):
                rows = got[0][torch.from_numpy(t.astype(np.int64)).cuda()].cpu().transpose(1, 2).reshape(-1, nkv * hd)
                rows = rows[length - m:length].view(torch.int16).numpy().view(np.uint16)
                assert np.array_equal(rows, want[length - m:length]), style
            at += m


def test_bounds_follow_rows_written_again_and_leave_nan_out():
    c = append_case("f16", (4, 2, 64), 32, [(3, 40)], False, 0, 0, True)
    k = c.nk.clone()
    k *= 100
    c.att.append(0, c.batch, c.q.cuda(), k.cuda(), c.nv.cuda())
    check_bounds(c)
    k[1, 3], k[2, 5], k[2, 6] = float("nan"), float("inf"), float("-inf")
    c.att.append(0, c.batch, c.q.cuda(), k.cuda(), c.nv.cuda())
    check_bounds(c)
    c.att.append(0, c.batch, c.q.cuda(), torch.zeros_like(k).cuda(), c.nv.cuda())
    check_bounds(c)
    c.batch.set([2], [39], c.tables)  # a rejected token: the page ends earlier
    c.att.append(0, c.batch, c.q[:2].cuda(), c.nk[:2].cuda(), c.nv[:2].cuda())
    c.n_new, c.lengths = [2], [39]
    check_bounds(c)


# ---- attention with a page budget ----

def sparse_case(kind, shape, page, seqs, seed=31, ties=False):
    heads, kv, d = shape
    n_pages = sum(-(-length // page) for _, length in seqs) + 2
    kb = torch.zeros((n_pages, kv, 2, d), dtype=torch.int8, device="cuda")
    ks = torch.zeros((n_pages, kv), device="cuda")
    c = Cache(kind, shape, page, seqs, seed=seed, key_bounds=kb, key_scales=ks)
    b, s = np.zeros((n_pages, kv, 2, d), np.int8), np.zeros((n_pages, kv), np.float32)
    for length, t in zip(c.lengths, c.tables):
        for j, p in enumerate(t):
            for h in range(kv):
                b[p, h], s[p, h] = R.bounds(c.k[0, p, h, :min(page, length - j * page)].double().numpy())
                if ties:  # few different pages, so that most scores are met many times
                    b[p, h], s[p, h] = (b[c.tables[0][j % 3], h], s[c.tables[0][j % 3], h]) if j >= 3 else (b[p, h], s[p, h])
    kb.copy_(torch.from_numpy(b))
    ks.copy_(torch.from_numpy(s))
    c.b, c.s = b, s
    return c


def check_sparse(c, select, first, last, q=None):
    q = c.q if q is None else q
    out, chosen = c.att.attend_sparse(0, c.batch, q.cuda(), select, first, last)
    out, chosen = out.double().cpu(), chosen.cpu().numpy()
    g, row = c.heads // c.kv, 0
    for m, length, t in zip(c.n_new, c.lengths, c.tables):
        for i in range(m):
            pos = length - m + i
            for h in range(c.kv):
                qh = q[row].view(c.kv, g, c.d)[h]
                want = R.choose(qh, pos // c.page, c.b[t, h], c.s[t, h], select, first, last)
                assert chosen[row, h].tolist() == want, (row, h, pos)
                at = torch.tensor([p * c.page + r for p in want if p >= 0 for r in range(c.page) if p * c.page + r <= pos])
                keys, values = (R.rows_of(x[0], t, h, length)[at] for x in (c.k, c.v))
                o, bound = R.attention(c.kind, qh, keys, values, torch.full((g,), len(at) - 1), c.d)
                near(out[row].view(c.kv, g, c.d)[h], o, bound, f"row {row} head {h}")
            row += 1


@pytest.mark.parametrize("kind,shape,page,seqs,budget", [
    ("f32", (16, 8, 128), 16, [(1, 1500), (1, 5), (0, 30), (1, 700)], (6, 1, 2)),
    ("bf16", (32, 8, 128), 64, [(1, 3000), (1, 640), (1, 64 * 9)], (8, 1, 2)),
    ("f16", (14, 2, 64), 16, [(21, 900), (1, 33), (3, 17)], (9, 2, 1)),
    ("bf16", (8, 2, 256), 32, [(1, 2000)], (4, 0, 1)),
    ("f32", (4, 4, 96), 128, [(5, 2000), (1, 1)], (3, 1, 1)),
    ("f16", (40, 2, 64), 16, [(1, 1000), (4, 500)], (16, 1, 3)),
    ("f16", (10, 2, 192), 16, [(1, 800)], (1, 0, 1)),
    ("bf16", (5, 1, 160), 16, [(2, 800)], (50, 3, 4))],
    ids=lambda x: "x".join(map(str, x)) if isinstance(x, tuple) else None)
def test_attend_sparse(kind, shape, page, seqs, budget):
    check_sparse(sparse_case(kind, shape, page, seqs), *budget)


@pytest.mark.parametrize("budget", [(7, 1, 1), (64, 0, 1), (200, 2, 2), (3, 1, 2)])
def test_equal_scores_take_the_lower_page(budget):
    check_sparse(sparse_case("f16", (4, 2, 64), 16, [(1, 16 * 300 + 5), (2, 1000)], ties=True), *budget)


def test_zero_and_large_queries_choose_as_defined():
    c = sparse_case("f32", (4, 2, 64), 16, [(4, 800)])
    q = c.q.clone()
    q[0], q[1], q[2] = 0, q[1] * 1e-9, q[2] * 1e9
    g, (out, chosen) = 2, c.att.attend_sparse(0, c.batch, q.cuda(), 8, 1, 2)
    for row in range(4):
        for h in range(2):
            want = R.choose(q[row].view(2, g, 64)[h], (796 + row) // 16, c.b[c.tables[0], h], c.s[c.tables[0], h], 8, 1, 2)
            assert chosen[row, h].tolist() == want


def test_many_pages_of_one_sequence():
    # 1 token behind 40000 positions in 2500 pages
    check_sparse(sparse_case("bf16", (4, 1, 64), 16, [(1, 40000)]), 100, 1, 2)


@pytest.mark.parametrize("kind,shape,page,length,select", [
    ("f16", (2, 1, 256), 16, 20000, 40), ("f32", (4, 2, 192), 16, 17000, 5), ("bf16", (8, 1, 128), 16, 40000, 300)])
def test_long_lists_of_single_tokens(kind, shape, page, length, select):
    # more pages than a wave lists, at the head sizes whose workgroups have two waves and four: with a second
    # sequence, and with so many pages and so few columns that these are shared out
    check_sparse(sparse_case(kind, shape, page, [(1, length), (1, 700)]), select, 1, 2)


def test_budgets_and_lists_beyond_one_workgroup():
    # more chosen pages than a fused workgroup holds, and more pages than its tiles leave room for
    check_sparse(sparse_case("f16", (2, 1, 64), 16, [(1, 16 * 2600 + 3), (1, 90)]), 2100, 1, 2)
    check_sparse(sparse_case("bf16", (2, 1, 64), 16, [(1, 16 * 16500)]), 20, 1, 2)


def test_layers_have_their_own_pages_and_bounds():
    # the same tokens in layers 0 and 2 of three, other ones in layer 1
    att = PagedAttention(3, 60, 16, 8, 2, 64, dtype="f16", rope_base=1e4, max_pos=600, bounds=True)
    batch = att.batch(2, 650, 600)
    rng = np.random.default_rng(3)
    tables = R.page_lists(rng, [500, 120], 16, 60)
    batch.set([500, 120], [500, 120], tables)
    g = torch.Generator(device="cuda").manual_seed(5)
    x = [[torch.randn(620, n * 64, generator=g, device="cuda").half() for n in (8, 2, 2)] for _ in range(2)]
    att.set_qk_norm(1, np.full(64, 2.0), np.full(64, 0.5))
    outs = []
    for layer in (0, 1, 2):
        q = att.append(layer, batch, *x[layer % 2])
        outs.append((q, att.attend(layer, batch, q), *att.attend_sparse(layer, batch, q, 5)))
    for a, b, c in zip(*outs):
        assert torch.equal(a, c) and not torch.equal(a, b)
    for t in (att.key_pages, att.val_pages, att.key_bounds, att.key_scales):
        assert torch.equal(t[0], t[2]) and not torch.equal(t[0], t[1])


def test_pages_listed_again_and_again():
    # a list may name a page that is only read many times: more of them than a choice can be made of
    c = sparse_case("f16", (2, 1, 64), 16, [(1, 16 * 40 + 1)])
    table = np.concatenate([np.tile(c.tables[0][:40], 820), c.tables[0][40:41]])
    n = 16 * 820 * 40 + 1
    batch = c.att.batch(1, 1, n)
    batch.set([1], [n], table[None])
    keys, values = (R.rows_of(x[0], table, 0, n) for x in (c.k, c.v))
    q = c.q.view(2, 64)
    near(c.att.attend(0, batch, c.q.cuda()).view(2, 64), *R.attention("f16", q, keys, values, torch.tensor([n - 1, n - 1]), 64))
    with pytest.raises(PQAError, match="32768"):
        c.att.attend_sparse(0, batch, c.q.cuda(), 8)
    batch.set([1], [16 * 32767 + 1], np.concatenate([table[:32767], table[-1:]])[None])
    out, chosen = c.att.attend_sparse(0, batch, c.q.cuda(), 8)
    assert torch.isfinite(out).all() and chosen[0, 0, -1] == 32767 and bool((chosen[0, 0, 1:] > chosen[0, 0, :-1]).all())


@pytest.mark.parametrize("shape", [(34, 2, 64), (34, 1, 128), (8, 2, 128)], ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("seqs", [[(1, 1500), (1, 900)], [(12, 700), (1, 900)]], ids=["tokens", "chunk"])
def test_attend_sparse_in_place(shape, seqs):
    # out is q, also where a KV head's query heads take several workgroups
    c = sparse_case("f16", shape, 16, seqs)
    want, chosen = c.att.attend_sparse(0, c.batch, c.q.cuda(), 6, 1, 2)
    for _ in range(5):
        q = c.q.cuda()
        out, again = c.att.attend_sparse(0, c.batch, q, 6, 1, 2, out=q)
        assert out is q and torch.equal(out, want) and torch.equal(again, chosen)


def test_infinities_among_chosen_pages():
    for kind in ("f32", "bf16"):
        c = sparse_case(kind, (8, 2, 128), 16, [(1, 900), (5, 700)])
        for t, at in zip(c.tables, (899, 698)):  # pages that are always chosen: the token's own, and one that three see
            c.v[0, t[at // 16], 0, at % 16, 7] = float("inf")
        c.dv.copy_(c.v)
        got, chosen = c.att.attend_sparse(0, c.batch, c.q.cuda(), 8, 1, 2)
        got = got.double().cpu().view(c.n, 2, 4, 128)
        for row in range(c.n):
            sees = row == 0 or 695 + row - 1 >= 698
            assert torch.isfinite(got[row, 1]).all()
            assert bool(torch.isinf(got[row, 0, :, 7]).all()) == sees and torch.isfinite(got[row, 0, :, :7]).all()


# ---- a run of them, as a server uses them ----

def test_a_server_step_by_step_against_the_contiguous_cache():
    # two requests: prompts in one batch, then three steps of a token each, with projections before and after;
    # the same through a contiguous context of each
    nh, nkv, hd, n_embd, base = 4, 2, 64, 512, 1e6
    rng = np.random.default_rng(5)

    def weights(rows, width):
        return (rng.standard_normal((rows, width)) / width ** 0.5).astype(np.float32).view(np.uint8)

    ws = [weights(r * hd, n_embd) for r in (nh, nkv, nkv)]
    wo = weights(n_embd, nh * hd)
    prompts, smax = (45, 70), 96
    with_proj = []
    for _ in range(3):
        a = PicoAttention(1, smax, nh, nkv, hd, rope_base=base)
        a.set_qkv_weights(0, n_embd, ws[0], 1, ws[1], 1, ws[2], 1)
        a.set_out_weights(0, n_embd, wo, 1)
        with_proj.append(a)
    proj, alone = with_proj[0], with_proj[1:]
    att = PagedAttention(1, 16, 16, nh, nkv, hd, dtype="f32", rope_base=base, max_pos=smax, bounds=True)
    batch = att.batch(2, sum(prompts))
    free = list(rng.permutation(16))
    tables = [[], []]
    lengths = [0, 0]
    for new in (prompts, (1, 1), (1, 1), (1, 1)):
        for i, m in enumerate(new):
            lengths[i] += m
            while len(tables[i]) * 16 < lengths[i]:
                tables[i].append(int(free.pop()))
        batch.set(list(new), lengths, tables)
        xb = torch.from_numpy(rng.standard_normal((sum(new), n_embd)).astype(np.float32)).cuda()
        x = torch.zeros_like(xb)
        q, k, v = proj.qkv_project_batch(0, xb)
        o = att.forward(0, batch, q, k, v)
        proj.out_project_batch(0, o, x)
        sparse, _ = att.attend_sparse(0, batch, att.append(0, batch, q, k, v), 8)
        want, row = torch.zeros_like(xb), 0
        for a, m, length in zip(alone, new, lengths):
            a.prefill_block(0, length - m, xb[row:row + m].contiguous(), want[row:row + m])
            row += m
        torch.cuda.synchronize()
        # the contiguous prefill's weights are rounded to fp16 (2^-11 of outputs around 0.3)
        assert float((x - want).abs().max()) <= 2e-3
        assert float((sparse - o).abs().max()) <= 1e-5  # every page is within the budget
    for i, a in enumerate(alone):
        kc, vc = a.kv_download(0, 0, lengths[i])
        for pages, rows in ((att.key_pages, kc), (att.val_pages, vc)):
            got = pages[0][torch.tensor(tables[i]).cuda()].cpu().transpose(1, 2).reshape(-1, nkv * hd)[:lengths[i]]
            assert np.array_equal(got.view(torch.int16).numpy().view(np.uint16), rows)


@pytest.mark.parametrize("rows,shape", [(64, (8, 2, 128)), (8, (8, 2, 128)), (8, (4, 1, 128))], ids=["chunks", "tokens", "shared"])
def test_captured_steps_follow_later_sets(rows, shape):
    # one graph of append, attention and attention with a budget; then other lengths, pages and sequences, chunks too;
    # for a batch of single tokens (which choose and attend in one launch), and one of long lists and few columns
    kind, page = "bf16", 16
    heads, kv, _ = shape
    top = 20000 if kv == 1 else 3000
    n_pages = top // page + 220
    cos, sin = rope_table(1e4, 128, top)
    att = PagedAttention(1, n_pages, page, *shape, dtype=kind, rope_cos=cos, rope_sin=sin, bounds=True)
    g = torch.Generator(device="cuda").manual_seed(3)
    for x in (att.key_pages, att.val_pages):
        x.copy_(torch.randn(x.shape, generator=g, device="cuda"))
    batch = att.batch(8, rows, top)
    q, k, v = (torch.zeros(rows, n * 128, dtype=torch.bfloat16, device="cuda") for n in (heads, kv, kv))
    out, sparse = torch.zeros_like(q), torch.zeros_like(q)
    turned = torch.zeros_like(q)
    chosen = torch.zeros((rows, kv, 6), dtype=torch.int32, device="cuda")

    def step():
        att.append(0, batch, q, k, v, q_out=turned)
        att.attend(0, batch, turned, out=out)
        att.attend_sparse(0, batch, turned, 6, 1, 2, out=sparse, chosen=chosen)

    rng = np.random.default_rng(1)

    def fill(seqs):
        batch.set([n for n, _ in seqs], [length for _, length in seqs], R.page_lists(rng, [length for _, length in seqs], page, n_pages))
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, generator=g, device="cuda"))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        fill([(1, 100), (1, 900)])
        step()
        torch.cuda.synchronize()
        graph = Graph(s.cuda_stream, step)
        for seqs in ([(1, 101), (1, 901)], [(1, 7)], [(1, 2900), (1, 1), (1, 450), (1, 17)], [(40, 300), (1, 1500), (20, 20)], [],
                     [(0, 50), (3, 2500)], [(1, 100)] * 8, [(1, top)]):
            if sum(m for m, _ in seqs) > rows:
                seqs = [(min(m, 1), length) for m, length in seqs]
            fill(seqs)
            n = sum(m for m, _ in seqs)
            for x in (out, sparse, turned):
                x.fill_(7)
            chosen.fill_(-7)
            kp, vp = att.key_pages.clone(), att.val_pages.clone()
            graph.launch(s.cuda_stream)
            got = [x.clone() for x in (turned, out, sparse, chosen, att.key_pages, att.val_pages, att.key_bounds)]
            assert all(bool((x[n:] == (-7 if x.dtype == torch.int32 else 7)).all()) for x in got[:4])
            att.key_pages.copy_(kp)
            att.val_pages.copy_(vp)
            step()
            torch.cuda.synchronize()
            for a, b, what in zip(got, (turned, out, sparse, chosen, att.key_pages, att.val_pages, att.key_bounds),
                                  ("q", "out", "sparse", "chosen", "K", "V", "bounds")):
                assert torch.equal(a, b), (seqs, what)
        with pytest.raises(PQAError, match="captured"):
            Graph(s.cuda_stream, lambda: batch.set([1], [5], [[0]]))
        with pytest.raises(PQAError, match="captured"):
            att.set_rope(0, 128, None, None, cos, sin)
        graph.close()
    torch.cuda.current_stream().wait_stream(s)
    gc.collect()  # the graphs whose capture failed leave no error behind
    assert float(torch.ones(3, device="cuda").sum()) == 3


def test_two_batches_on_two_streams():
    c = Cache("bf16", (32, 8, 128), 32, [(1, 6000), (1, 500)], seed=41)
    q = c.q.cuda()
    other = c.att.batch(1, 1)
    other.set([1], [6000], [c.tables[0]])
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    outs = []
    for _ in range(10):
        with torch.cuda.stream(a):
            outs.append((c.att.attend(0, c.batch, q), 2))
        with torch.cuda.stream(b):
            outs.append((c.att.attend(0, other, q[:1]), 1))
    torch.cuda.synchronize()
    want, bound = c.want()
    for o, n in outs:
        near(o, want[:n], bound[:n])


def test_sets_while_calls_run():
    # the batch is set again and again without a wait between: each call uses what it was set to before it
    c = Cache("f16", (16, 8, 128), 16, [(1, 3000), (1, 40), (30, 500)], seed=43)
    q = c.q.cuda()
    want, bound = c.want()
    views = [([1, 1, 30], slice(0, 32)), ([1, 0, 0], slice(0, 1)), ([0, 1, 0], slice(1, 2)), ([0, 0, 30], slice(2, 32))]
    outs = []
    for i in range(24):
        n_new, rows = views[i % 4]
        c.batch.set(n_new, c.lengths, c.tables)
        outs.append((c.att.attend(0, c.batch, q[rows]), rows))
    for o, rows in outs:
        near(o, want[rows], bound[rows])


# ---- refusals that need a handle ----

def test_refusals():
    c = append_case("bf16", (8, 2, 128), 16, [(1, 30), (4, 20)], False, 0, 128, False)
    q, k, v = c.q.cuda(), c.nk.cuda(), c.nv.cuda()
    before = c.dk.clone()
    for call, match in [
            (lambda: c.att.attend(1, c.batch, q), "layer"), (lambda: c.att.attend(-1, c.batch, q), "layer"),
            (lambda: c.att.attend_sparse(0, c.batch, q, 4), "bounds"),
            (lambda: c.att.attend(0, c.att.batch(2, 5), q), "holds nothing"),
            (lambda: c.batch.set([1], [36], [[0, 1, 2]]), "rotation"),
            (lambda: c.batch.set([1], [30], [[0, c.n_pages]]), "page"),
            (lambda: c.batch.set([6], [30], [[0, 1]]), "new tokens"),
            (lambda: c.batch.set([1, 1], [3, 3], [[0], [0]]), "listed twice"),
            (lambda: c.att.batch(0, 5), "positive"), (lambda: c.att.batch(1, 5, -1), "positive"),
            (lambda: c.att.set_qk_norm(0, np.ones(128), None), "both"), (lambda: c.att.set_qk_norm(3, np.ones(128), np.ones(128)), "layer"),
            (lambda: PagedAttention(1, 4, 24, 8, 2, 128), "page_size"), (lambda: PagedAttention(1, 4, 16, 8, 3, 128), "multiple"),
            (lambda: PagedAttention(1, 4, 16, 8, 2, 80), "head_dim")]:
        with pytest.raises(PQAError, match=match):
            call()
    for call in [lambda: c.att.attend(0, c.batch, q[:4]), lambda: c.att.attend(0, c.batch, q.float()),
                 lambda: c.att.attend(0, c.batch, q.cpu()), lambda: c.att.attend(0, c.batch, q[:, :64]),
                 lambda: c.att.attend(0, c.batch, q.t().contiguous().t()), lambda: c.att.attend(0, c.batch, q, out=q[:3]),
                 lambda: c.att.attend(0, c.batch, q, out=q[:1].expand(5, -1)), lambda: c.att.append(0, c.batch, q, k[:4], v),
                 lambda: c.att.append(0, c.batch, q, k, v.float()), lambda: c.batch.set([1.5], [3], [[0]]),
                 lambda: c.batch.set([1, 1], [3], [[0], [1]]), lambda: c.batch.set([1], [3], [[0], [1]]),
                 lambda: c.att.set_rope(0, 128, rope_cos=np.zeros((4, 3)), rope_sin=np.zeros((4, 3)))]:
        with pytest.raises(ValueError):
            call()
    torch.cuda.synchronize()
    assert torch.equal(c.dk.view(torch.int16), before.view(torch.int16))
    # a refused set leaves the batch as it was
    near(c.att.attend(0, c.batch, q), *c.want())
    other = PagedAttention(1, 4, 16, 8, 2, 128, dtype="bf16")
    with pytest.raises(PQAError, match="another handle"):
        other.attend(0, c.batch, q)
    s = sparse_case("f16", (4, 2, 64), 16, [(1, 100)])
    for budget in [(0, 0, 1), (4, -1, 2), (4, 1, 0), (4, 3, 2)]:
        with pytest.raises((PQAError, ValueError)):
            s.att.attend_sparse(0, s.batch, s.q.cuda(), *budget)
    # a changed rotation is met by a batch that was checked against the old one, also after a refused set
    c.att.set_rope(0, 128, 1e4, 30)
    for _ in range(2):
        with pytest.raises(PQAError, match="set the batch again"):
            c.att.append(0, c.batch, q, k, v)
        with pytest.raises(PQAError, match="rotation"):
            c.batch.set([1], [31], [[0, 1]])
    c.batch.set(c.n_new, c.lengths, c.tables)
    c.att.append(0, c.batch, q, k, v)


def test_a_closed_cache_and_its_batches():
    c = Cache("f16", (4, 2, 64), 16, [(1, 30)], seed=1)
    c.att.close()
    for call in (lambda: c.att.attend(0, c.batch, c.q.cuda()), lambda: c.batch.set([1], [30], c.tables)):
        with pytest.raises(RuntimeError, match="destroyed"):
            call()
    c.batch.close()
    d = Cache("f16", (4, 2, 64), 16, [(1, 30)], seed=1)
    d.batch.close()
    with pytest.raises(RuntimeError, match="destroyed"):
        d.att.attend(0, d.batch, d.q.cuda())


def test_calls_run_on_the_current_stream():
    # behind a long copy on a side stream, which the default stream does not wait for
    c = Cache("bf16", (8, 2, 128), 16, [(1, 500), (30, 90)], seed=3)
    want, bound = c.want()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    big = torch.empty(1 << 28, dtype=torch.uint8, device="cuda")
    with torch.cuda.stream(s):
        for _ in range(4):
            big.add_(1)
        q = torch.empty_like(c.q, device="cuda")
        q.copy_(c.q)
        out = c.att.attend(0, c.batch, q)
        got = out.cpu()
    near(got, want, bound)


def test_an_empty_batch_launches_nothing():
    c = Cache("f32", (4, 2, 64), 16, [(0, 30), (0, 0)], seed=1)
    q = torch.zeros(0, 256, device="cuda")
    assert c.att.attend(0, c.batch, q).shape == (0, 256)
    c.batch.set([], [], [])
    assert c.att.attend(0, c.batch, q).shape == (0, 256)
    wide = torch.full((3, 256), 2.0, device="cuda")
    assert bool((c.att.attend(0, c.batch, wide, out=wide) == 2).all())
