"""The draft-verification operators on the B200 against plain 64-bit forms in numpy.

Tolerances count roundings. bf16 rounds by at most 2^-8 of the value, fp32 by 2^-24; each test
states what its operator rounds and bounds every element by that.
"""
import ctypes as C

import numpy as np
import pytest

import k3cuda
import workloads as W

pytestmark = pytest.mark.gpu

BF, F4 = 2.0 ** -8, 2.0 ** -24
NAN16 = 0x7FC0


class Paged:
    """A paged cache and a batch of new tokens. Rows that no sequence owns, and the rows of the
    new tokens until they are written, hold NaN."""

    def __init__(self, ctx, rng, lens, toks, page, pad=0, spare=2):
        self.ctx, self.lens, self.toks, self.page = ctx, list(lens), list(toks), page
        B = len(lens)
        need = [-(-(ln + t) // page) for ln, t in zip(lens, toks)]
        self.n_pages = sum(need) + spare
        self.width = max(1, max(need)) + 1
        perm = rng.permutation(self.n_pages).astype(np.int32)
        self.table = np.full((B, self.width), -7, np.int32)   # entries past a sequence: unused
        at = 0
        for b, k in enumerate(need):
            self.table[b, :k] = perm[at:at + k]
            at += k
        self.cu = np.concatenate([[0], np.cumsum(toks)]).astype(np.int32)
        self.T = int(self.cu[-1]) + pad
        self.latent = np.full((self.n_pages * page, 512), NAN16, np.uint16)
        self.rope = np.full((self.n_pages * page, 64), NAN16, np.uint16)
        for b, ln in enumerate(lens):
            r = self.rows(b)[:ln]
            self.latent[r] = W.f32_to_bf16(rng.standard_normal((ln, 512)).astype(np.float32) * 0.5)
            self.rope[r] = W.f32_to_bf16(rng.standard_normal((ln, 64)).astype(np.float32))
        self.up()

    def rows(self, b):
        p = np.arange(self.lens[b] + self.toks[b])
        return self.table[b, p // self.page].astype(np.int64) * self.page + p % self.page

    def up(self):
        c = self.ctx
        self.d = [c.upload(self.latent), c.upload(self.rope), c.upload(self.table),
                  c.upload(np.asarray(self.lens, np.int32)), c.upload(self.cu)]
        self.cache = k3cuda.PagedCache(latent=self.d[0].ptr, rope=self.d[1].ptr,
                                       page_table=self.d[2].ptr, n_pages=self.n_pages,
                                       page_size=self.page, max_pages=self.width)
        self.batch = k3cuda.TokenBatch(ctx_lens=self.d[3].ptr, cu_tokens=self.d[4].ptr,
                                       B=len(self.lens), T=self.T)

    def fill_drafts(self, rng):
        """The new tokens' rows, as an append would leave them."""
        for b, ln in enumerate(self.lens):
            r = self.rows(b)[ln:]
            self.latent[r] = W.f32_to_bf16(rng.standard_normal((len(r), 512)).astype(np.float32))
            self.rope[r] = W.f32_to_bf16(rng.standard_normal((len(r), 64)).astype(np.float32))
        self.up()


# offsets of three sequences in eight token rows, and how many of the sequences are in order
OUT_OF_ORDER = [([0, 5, -4, 8], 1), ([0, 2, 1, 8], 1), ([0, 2, 5, 4], 2), ([0, 3, 9, 8], 1),
                ([-1, 2, 5, 8], 0), ([0, 8, 3, 5], 1), ([2, 4, 4, 3], 2), ([0, 3, 2000000000, 8], 1),
                ([0, 4, 6, 2000000000], 2), ([1, 0, 4, 8], 0)]


def reports(ctx, text):
    """The next sync reports a bad table."""
    try:
        ctx.sync()
    except k3cuda.K3CudaError as e:
        assert e.code == k3cuda.ERR_ARG and text in str(e), e
    else:
        pytest.fail("nothing reported")


def out_of_order(ctx, rng, cu, good):
    toks = [max(0, min(cu[b + 1] - cu[b], 8)) if b < good else 4 for b in range(3)]
    p = Paged(ctx, rng, [20, 30, 10], toks, 16)
    p.fill_drafts(rng)
    p.cu, p.T = np.array(cu, np.int32), 8
    p.up()
    return p


# ------------------------------------------------------------------------------- append
def rotated(x, pos, inv_freq, style):
    """R_p x in 64 bits, and a bound of what fp32 rotation may be off: the angle's reduction
    (2^-52 of it) and its rounding to fp32 (pi 2^-24), two ulp of the sine and cosine, two
    products and a sum, each relative to |x0| + |x1|."""
    if inv_freq is None:
        return x, np.zeros_like(x)
    a = pos.astype(np.float64)[:, None] * inv_freq.astype(np.float64)
    for _ in range(x.ndim - 2):
        a = a[:, None]
    c, s = np.cos(a), np.sin(a)
    i = np.arange(32)
    i0, i1 = (i, i + 32) if style == k3cuda.ROPE_HALF else (2 * i, 2 * i + 1)
    y, e = np.empty_like(x), np.empty_like(x)
    x0, x1 = x[..., i0], x[..., i1]
    y[..., i0], y[..., i1] = x0 * c - x1 * s, x0 * s + x1 * c
    off = (np.abs(x0) + np.abs(x1)) * (np.abs(a) * 2.0 ** -51 + (np.pi + 2 * 2 + 3) * F4)
    e[..., i0] = e[..., i1] = off
    return y, e


def near(got16, want, extra=0.0):
    got = W.bf16_to_f32(got16).astype(np.float64)
    lim = BF * np.abs(want) * (1 + 8 * F4) + 8 * F4 * np.abs(want) + extra + 1e-38
    bad = ~(np.abs(got - want) <= lim)
    assert not bad.any(), (np.argwhere(bad)[:4], got[bad][:4], want[bad][:4])


def run_append(ctx, rng, p, H, io, style, positions=True, freq=True, extra_stride=0, null_q=False):
    bf16 = io == k3cuda.BF16
    T, tot = p.T, int(p.cu[-1])
    cs, qs = 576 + extra_stride, H * 192 + extra_stride
    ct = rng.standard_normal((T, cs)).astype(np.float32)
    q = rng.standard_normal((T, max(qs, 8))).astype(np.float32)
    if bf16:
        ct, q = W.round_bf16(ct), W.round_bf16(q)
    conv = W.f32_to_bf16 if bf16 else (lambda a: a)
    w = (1 + 0.1 * rng.standard_normal(512)).astype(np.float32)
    inv = (50000.0 ** (-np.arange(0, 64, 2) / 64)).astype(np.float32)
    pos = rng.integers(0, 1 << 30, T).astype(np.int32)
    dct, dq, dw, dinv, dpos = (ctx.upload(a) for a in (conv(ct), conv(q), w, inv, pos))
    qn, qr = ctx.upload(np.full((T, max(H, 1), 128), 0x1234, np.uint16)), ctx.upload(
        np.full((T, max(H, 1), 64), 0x1234, np.uint16))
    ctx.mla_paged_append(p.cache, p.batch, dct, dw, 1e-6, q=None if null_q else dq, q_nope=qn,
                         q_rope=qr, H=H, positions=dpos if positions else None,
                         inv_freq=dinv if freq else None, rope_style=style, io_dtype=io,
                         ct_stride=cs, q_stride=qs)
    ctx.sync()
    where = np.concatenate([p.lens[b] + np.arange(t) for b, t in enumerate(p.toks)]).astype(np.int64)
    at = pos[:tot] if positions else where
    f = inv if freq else None
    c = ct[:tot].astype(np.float64)
    lat = c[:, :512] / np.sqrt((c[:, :512] ** 2).mean(-1, keepdims=True) + np.float64(
        np.float32(1e-6))) * w
    key, key_off = rotated(c[:, 512:576], at, f, style)
    row = np.concatenate([p.rows(b)[p.lens[b]:] for b in range(len(p.lens))])
    got_l, got_r = p.d[0].numpy(), p.d[1].numpy()
    near(got_l[row], lat)
    near(got_r[row], key, key_off)
    rest = np.ones(len(got_l), bool)
    rest[row] = False
    assert (got_l[rest] == p.latent[rest]).all() and (got_r[rest] == p.rope[rest]).all()
    gn, gr = qn.numpy(), qr.numpy()
    if H:
        qq = q[:tot, :H * 192].reshape(tot, H, 192).astype(np.float64)
        near(gn[:tot], qq[..., :128])
        near(gr[:tot], *rotated(qq[..., 128:], at, f, style))
    if not H:
        tot = 0
    assert (gn[tot:] == 0x1234).all() and (gr[tot:] == 0x1234).all()   # padding rows


@pytest.mark.parametrize("io", [k3cuda.F32, k3cuda.BF16])
@pytest.mark.parametrize("style", [k3cuda.ROPE_HALF, k3cuda.ROPE_INTERLEAVED])
@pytest.mark.parametrize("H,page,lens,toks,pad", [
    (16, 64, [100], [1], 0),
    (1, 8, [0, 7, 8, 9, 300], [1, 9, 0, 64, 3], 5),
    (17, 16, [31, 0, 0, 1000], [0, 0, 40, 2], 1),
    (128, 32, [5, 64], [33, 31], 0),
    (0, 128, [127, 128], [1, 2], 3),
])
def test_append(ctx, io, style, H, page, lens, toks, pad):
    rng = np.random.default_rng([io, style, H, page])
    run_append(ctx, rng, Paged(ctx, rng, lens, toks, page, pad), H, io, style, null_q=H == 0)


def test_append_variants(ctx):
    """No rotation, the cache position as rotation position, rows with a stride, and 70 sequences
    (more than two rounds of the offset search)."""
    rng = np.random.default_rng(5)
    for kw in (dict(freq=False), dict(positions=False), dict(extra_stride=8)):
        for io in (k3cuda.F32, k3cuda.BF16):
            p = Paged(ctx, rng, [40, 3, 0], [5, 0, 70], 16, 2)
            run_append(ctx, rng, p, 12, io, k3cuda.ROPE_HALF, **kw)
    toks = rng.integers(0, 4, 1100)
    p = Paged(ctx, rng, rng.integers(0, 30, 1100), toks, 8, 1)
    run_append(ctx, rng, p, 2, k3cuda.F32, k3cuda.ROPE_INTERLEAVED)


def test_append_reports_bad_tables(ctx):
    """A bad sequence is left out, the others are written, the next sync says so once."""
    rng = np.random.default_rng(6)
    ct, w = rng.standard_normal((8, 576)).astype(np.float32), np.ones(512, np.float32)
    dct, dw = ctx.upload(ct), ctx.upload(w)
    for what, text in (("page", "outside the cache"), ("len", "negative length"),
                       ("table", "page table"), ("cu", "cu_tokens|outside the cache")):
        p = Paged(ctx, rng, [20, 30, 10], [2, 3, 3], 16)
        if what == "page":
            p.table[1, 30 // 16] = p.n_pages
            p.table[1, 32 // 16] = -1
        if what == "len":
            p.lens[1] = -1
        if what == "table":
            p.lens[1] = p.width * 16 - 2
        if what == "cu":
            p.cu = np.array([0, 2, 1, 8], np.int32)   # sequence 1 falls; 2 has seven rows
        p.up()
        ctx.mla_paged_append(p.cache, p.batch, dct, dw, 1e-6)
        with pytest.raises(k3cuda.K3CudaError, match=text) as e:
            ctx.sync()
        assert e.value.code == k3cuda.ERR_ARG
        ctx.sync()   # reported once
        got = p.d[0].numpy()
        for b, (a, n) in enumerate(((0, 2), (2, 3), (5, 3))):
            if b == 1 or what == "cu":
                continue
            p.lens[b] = [20, 30, 10][b]
            want = ct[a:a + n, :512].astype(np.float64)
            want /= np.sqrt((want ** 2).mean(-1, keepdims=True) + 1e-6)
            near(got[p.rows(b)[p.lens[b]:]], want)


def test_append_offsets_at_any_alignment(ctx):
    """Offsets that begin anywhere in a 16-byte vector, more of them than a block reads at once."""
    rng = np.random.default_rng(17)
    for shift in range(4):
        for B in (1, 2, 5, 7, 530):
            p = Paged(ctx, rng, rng.integers(0, 30, B), rng.integers(0, 4, B), 8, 1)
            d = ctx.upload(np.concatenate([np.full(shift, -5), p.cu, [-5] * 4]).astype(np.int32))
            p.batch.cu_tokens = d.ptr + 4 * shift
            run_append(ctx, rng, p, 1, k3cuda.F32, k3cuda.ROPE_HALF)


@pytest.mark.parametrize("cu,good", OUT_OF_ORDER)
def test_append_offsets_out_of_order(ctx, cu, good):
    """Sequences before the first offset that is out of order are appended; nothing else changes."""
    rng = np.random.default_rng(14)
    p = out_of_order(ctx, rng, cu, good)
    ct, w = rng.standard_normal((8, 576)).astype(np.float32), np.ones(512, np.float32)
    q = rng.standard_normal((8, 3, 192)).astype(np.float32)
    dct, dw, dq = ctx.upload(ct), ctx.upload(w), ctx.upload(q)
    qn, qr = (ctx.upload(np.full((8, 3, n), 0x1234, np.uint16)) for n in (128, 64))
    ctx.mla_paged_append(p.cache, p.batch, dct, dw, 1e-6, q=dq, q_nope=qn, q_rope=qr, H=3)
    reports(ctx, "cu_tokens")
    lat, rope, gn, gr = p.d[0].numpy(), p.d[1].numpy(), qn.numpy(), qr.numpy()
    rest, told = np.ones(len(lat), bool), np.zeros(8, bool)
    for b in range(good):
        t, row = slice(cu[b], cu[b + 1]), p.rows(b)[p.lens[b]:]
        c = ct[t].astype(np.float64)
        near(lat[row], c[:, :512] / np.sqrt((c[:, :512] ** 2).mean(-1, keepdims=True) + 1e-6))
        near(rope[row], c[:, 512:])
        near(gn[t], q[t, :, :128].astype(np.float64))
        near(gr[t], q[t, :, 128:].astype(np.float64))
        rest[row], told[t] = False, True
    assert (lat[rest] == p.latent[rest]).all() and (rope[rest] == p.rope[rest]).all()
    assert (gn[~told] == 0x1234).all() and (gr[~told] == 0x1234).all()


def test_each_bad_call_is_reported(ctx):
    """A call that follows a report at once is reported too, a good one is not."""
    rng = np.random.default_rng(18)
    p = Paged(ctx, rng, [20], [2], 16)
    bad = k3cuda.TokenBatch(ctx_lens=p.d[3].ptr, cu_tokens=p.d[4].ptr, B=1, T=1)   # the offsets pass T
    dct = ctx.upload(rng.standard_normal((2, 576)).astype(np.float32))
    dw = ctx.upload(np.ones(512, np.float32))
    for k in range(200):
        ctx.mla_paged_append(p.cache, bad, dct, dw, 1e-6)
        reports(ctx, "cu_tokens")
        if k % 2:
            ctx.mla_paged_append(p.cache, p.batch, dct, dw, 1e-6)
            ctx.sync()


# ------------------------------------------------------------------------- tree attention
def tree_words(rng, toks, kind):
    """Visibility words: `tree` random trees, `chain` every earlier draft, `none` nothing,
    `self` each draft itself only, `wild` any bits (bits past the drafts included)."""
    out = []
    for n in toks:
        w = []
        for i in range(n):
            if kind == "tree":
                par = int(rng.integers(max(-1, i - 3), i)) if i else -1
                w.append((w[par] if par >= 0 else 0) | (1 << i))
            elif kind == "chain":
                w.append((1 << (i + 1)) - 1)
            elif kind == "self":
                w.append(1 << i)
            elif kind == "wild":
                w.append(int(rng.integers(0, 1 << 32)) << 32 | int(rng.integers(0, 1 << 32)))
            else:
                w.append(0)
        out += w
    return np.array(out, np.uint64)


def tree_oracle(p, words, qn, qr, uk, uv, scale):
    """(out, bound) in 64 bits. The kernel rounds the absorbed query to bf16 (2^-8 of each of its
    elements, so a score moves by at most D_r = 2^-8 scale sum |qa_d c_rd|), each weight to bf16
    (2^-8 of it), and sums in fp32. With p_r the weights, log p_r moves by at most
    D_r + sum p D, so out moves by at most sum p_r (2^-8 + D_r + sum p D) |v_r| to first order;
    the factor 1.05 covers the second, fp32 sums 2^-16. These share their factor over the 512
    terms of v_r = W_UV c_r, which may cancel; the weighted sum of the c_r does not when it is
    summed in fp32 (n terms, n 2^-24), carried as two bf16 halves (2^-16) and multiplied by W_UV
    (512 terms): that adds (2^-16 + (n + 512) 2^-24) sum_r p_r |W_UV| |c_r|."""
    T, H = qn.shape[:2]
    out, lim = np.zeros((T, H, 128)), np.zeros((T, H, 128))
    for b, n in enumerate(p.toks):
        ln, t0 = p.lens[b], int(p.cu[b])
        rows, t = p.rows(b), slice(t0, t0 + n)
        c, r = (W.bf16_to_f32(a[rows]).astype(np.float64) for a in (p.latent, p.rope))
        see = np.array([[j < ln or (int(w) >> (j - ln)) & 1 for j in range(ln + n)]
                        for w in words[t]], bool).reshape(n, ln + n)
        some = see.any(-1)
        for h in range(H if some.any() else 0):
            qa = qn[t, h] @ uk[h]
            s = (qa @ c.T + qr[t, h] @ r.T) * scale
            D = BF * abs(scale) * (np.abs(qa) @ np.abs(c).T)
            s = np.where(see, s, -np.inf)
            top = np.where(some, s.max(-1), 0.0)
            e = np.exp(s - top[:, None])
            pr = e / np.where(some, e.sum(-1), 1.0)[:, None]
            v = c @ uv[h].T
            out[t, h] = pr @ v
            d = BF + D + (pr * D).sum(-1, keepdims=True) + 2.0 ** -16
            lim[t, h] = 1.05 * (pr * d) @ np.abs(v)
            lim[t, h] += (2.0 ** -16 + (ln + n + 512) * F4) * (pr @ np.abs(c)) @ np.abs(uv[h]).T
    return out, lim


def tree_inputs(ctx, rng, p, H):
    b = W.f32_to_bf16
    g = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
    return [b(g(p.T, H, 128)), b(g(p.T, H, 64)), b(g(H, 128, 512) * 0.04),
            b(g(H, 128, 512) * 0.04)]


def run_tree(ctx, p, x, words, H, scale, out_dtype=k3cuda.F32, ws=None):
    dx = [ctx.upload(a) for a in x]
    dm = None if words is None else ctx.upload(words if len(words) else np.zeros(1, np.uint64))
    fill = 0x4B4B if out_dtype == k3cuda.BF16 else 0x4B4B4B4B
    out = ctx.empty((p.T, H, 128), np.uint16 if out_dtype == k3cuda.BF16 else np.float32)
    out.fill(0x4B)
    n = ctx.mla_tree_attend_workspace(len(p.lens), p.T, H)
    if ws is None:
        ws = ctx.empty((max(n, 1),), np.uint8)
        ws.fill(0xFF)
    ctx.mla_tree_attend(out, dx[0], dx[1], p.cache, p.batch, dx[2], dx[3], H, scale, ws, n,
                        tree_mask=dm, out_dtype=out_dtype)
    ctx.sync()
    o = out.numpy()
    tail = o[int(p.cu[-1]):]
    assert (tail.view(np.uint16 if out_dtype == k3cuda.BF16 else np.uint32) == fill).all()
    return W.bf16_to_f32(o) if out_dtype == k3cuda.BF16 else o


def check_tree(ctx, rng, lens, toks, page, H, kind, out_dtype=k3cuda.F32, pad=0, scale=0.0722):
    p = Paged(ctx, rng, lens, toks, page, pad)
    p.fill_drafts(rng)
    x = tree_inputs(ctx, rng, p, H)
    words = tree_words(rng, toks, kind)
    f = lambda a: W.bf16_to_f32(a).astype(np.float64)  # noqa: E731
    want, lim = tree_oracle(p, words, *(f(a) for a in x), scale)
    dev = np.concatenate([words, np.zeros(pad, np.uint64)])
    got = run_tree(ctx, p, x, None if kind == "chain" else dev, H, scale, out_dtype)
    if out_dtype == k3cuda.BF16:
        lim = lim + BF * (np.abs(want) + lim)
    tot = int(p.cu[-1])
    bad = ~(np.abs(got[:tot] - want[:tot]) <= lim[:tot] + 1e-30)
    assert not bad.any(), (np.argwhere(bad)[:3], bad.mean(), got[:tot][bad][:3],
                           want[:tot][bad][:3], lim[:tot][bad][:3])
    return p, x, dev, got


@pytest.mark.parametrize("H", [1, 12, 16, 96, 128])
@pytest.mark.parametrize("kind", ["tree", "chain", "wild"])
def test_tree_ragged(ctx, H, kind):
    rng = np.random.default_rng([H, len(kind)])
    check_tree(ctx, rng, [0, 1, 63, 64, 65, 200, 130, 0], [1, 3, 1, 0, 2, 5, 7, 4], 16, H, kind,
               pad=2)


@pytest.mark.parametrize("page", [8, 16, 32, 64, 128, 256])
def test_tree_pages(ctx, page):
    rng = np.random.default_rng(page)
    check_tree(ctx, rng, [page - 1, page, 3 * page + 5, 700], [2, 64, 9, 1], page, 3, "tree",
               k3cuda.BF16)


@pytest.mark.parametrize("len0", [74 * 128 - 1, 74 * 128])
def test_tree_a_tile_for_each_cluster_and_one_more(ctx, len0):
    rng = np.random.default_rng(len0)
    check_tree(ctx, rng, [len0], [1], 128, 16, "tree")


def test_tree_drafts_across_tiles(ctx):
    """Drafts that end one tile and begin the next, 32-row chunks without a row, with one, full."""
    rng = np.random.default_rng(21)
    check_tree(ctx, rng, [100, 127, 96, 31, 32, 33, 65], [60, 64, 33, 1, 32, 2, 63], 8, 6, "tree")


@pytest.mark.parametrize("busy", [40, 1500])
def test_tree_many_sequences(ctx, busy):
    """More sequences than the plan's block has threads, few of them or most with a token."""
    rng = np.random.default_rng(busy)
    B = 2300
    toks = np.zeros(B, int)
    toks[rng.permutation(B)[:busy]] = rng.integers(1, 3, busy)
    lens = np.where(rng.random(B) < 0.9, rng.integers(0, 20, B), rng.integers(100, 400, B))
    check_tree(ctx, rng, lens.tolist(), toks.tolist(), 8, 1, "tree", pad=1)


@pytest.mark.parametrize("lens,toks,page,H", [
    ([100] * 160, [29] * 160, 8, 4),                   # a full tile of drafts, then one of one row
    ([3 * 128 + 70, 2 * 128 - 1, 127] * 40, [64, 2, 33] * 40, 8, 2),
    ([12000, 128, 5 * 128], [3, 1, 64], 16, 24)])
def test_tree_tiles_past_the_cached_rows_wait_for_the_last(ctx, lens, toks, page, H):
    """Tiles with drafts behind cached tiles and behind one another, the chunks of the second with
    and without rows, row tile after row tile; the caches cold and warm, all with the same bits.
    Unwritten rows hold NaN."""
    rng = np.random.default_rng([len(lens), page, H])
    p, x, words, got = check_tree(ctx, rng, lens, toks, page, H, "tree")
    for k in range(12):
        if k % 2:
            ctx.flush_l2()
        again = run_tree(ctx, p, x, words, H, 0.0722)
        assert (again.view(np.uint32) == got.view(np.uint32)).all()


def test_tree_millions_of_empty_sequences(ctx):
    """As many sequences as a call takes; few of them have tokens, and lie far apart."""
    rng = np.random.default_rng(24)
    B, k = (1 << 24) - 1, 160
    p = Paged(ctx, rng, rng.integers(0, 250, k), rng.integers(1, 4, k), 256)   # a page each
    p.fill_drafts(rng)
    x = tree_inputs(ctx, rng, p, 2)
    words = tree_words(rng, p.toks, "tree")
    f = lambda a: W.bf16_to_f32(a).astype(np.float64)  # noqa: E731
    want, lim = tree_oracle(p, words, *(f(a) for a in x), 0.0722)
    at = np.arange(k) * (B // k) + rng.integers(0, B // k, k)
    lens, n, table = np.full(B, 7, np.int32), np.zeros(B, np.int64), np.full(B, -3, np.int32)
    lens[at], n[at], table[at] = p.lens, p.toks, p.table[:, 0]
    cu = np.concatenate([[0], np.cumsum(n)]).astype(np.int32)
    p.d[2:] = [ctx.upload(a) for a in (table, lens, cu)]
    p.cache.max_pages, p.cache.page_table = 1, p.d[2].ptr
    p.batch = k3cuda.TokenBatch(ctx_lens=p.d[3].ptr, cu_tokens=p.d[4].ptr, B=B, T=p.T)
    m = ctx.mla_tree_attend_workspace(B, p.T, 2)
    ws, out = ctx.empty((m,), np.uint8), ctx.empty((p.T, 2, 128), np.float32)
    dx, dw = [ctx.upload(a) for a in x], ctx.upload(words)
    ctx.mla_tree_attend(out, dx[0], dx[1], p.cache, p.batch, dx[2], dx[3], 2, 0.0722, ws, m,
                        tree_mask=dw)
    ctx.sync()
    assert (np.abs(out.numpy() - want) <= lim).all()


def test_tree_sees_nothing(ctx):
    rng = np.random.default_rng(8)
    *_, got = check_tree(ctx, rng, [0, 0, 5], [3, 1, 2], 16, 5, "none")
    assert (got[:4] == 0).all() and (got[4:] != 0).any()
    check_tree(ctx, rng, [0, 100], [64, 33], 32, 4, "self")


@pytest.mark.parametrize("B,n,H,ctx_len", [(1, 1, 16, 3000), (1, 1, 128, 40000), (1, 26, 12, 20011),
                                           (3, 64, 8, 1500), (40, 1, 16, 300), (2, 13, 128, 777)])
def test_tree_split_contexts(ctx, B, n, H, ctx_len):
    """Contexts cut over many blocks and joined; more than eight tokens and fewer."""
    rng = np.random.default_rng([B, n, H])
    lens = [max(0, ctx_len - 37 * b) for b in range(B)]
    check_tree(ctx, rng, lens, [n] * B, 64, H, "tree", k3cuda.BF16 if B > 2 else k3cuda.F32)


def test_tree_scores_far_apart(ctx):
    """Scores that grow by thousands along the context (the running maximum moves late), and a
    scale of zero and of either sign."""
    rng = np.random.default_rng(9)
    check_tree(ctx, rng, [300, 0], [3, 2], 16, 5, "tree", scale=0.0)
    for scale in (0.0722, -0.0722):
        p = Paged(ctx, rng, [500, 70], [4, 2], 16)
        p.fill_drafts(rng)
        for b in range(2):
            r = p.rows(b)
            p.rope[r] = W.f32_to_bf16(np.linspace(0, 300, len(r))[:, None].astype(np.float32) *
                                      np.ones((1, 64), np.float32))
        p.up()
        x = tree_inputs(ctx, rng, p, 6)
        x[1] = W.f32_to_bf16(np.full((p.T, 6, 64), 0.5, np.float32))
        words = tree_words(rng, p.toks, "tree")
        f = lambda a: W.bf16_to_f32(a).astype(np.float64)  # noqa: E731
        want, lim = tree_oracle(p, words, *(f(a) for a in x), scale)
        # scores of up to 700 are formed in fp32 from 576 products
        s_off = 576 * F4 * 700
        got = run_tree(ctx, p, x, words, 6, scale)
        big = np.abs(f(p.latent[np.concatenate([p.rows(0), p.rows(1)])])).max() * 512 * 0.2
        assert (np.abs(got - want) <= lim * (1 + 2 * s_off) + 2 * s_off * big * 1e-3).all()


def test_tree_hidden_rows_may_hold_anything(ctx):
    """Infinities and NaN in hidden draft rows, in unwritten rows and in other sequences' pages
    reach nobody; a visible one gives NaN to exactly those that see it."""
    rng = np.random.default_rng(10)
    H = 10
    for bad in (NAN16, 0x7F80, 0xFF80, 0x7FFF, 0xFFC0):
        p = Paged(ctx, rng, [70, 20], [9, 5], 16)
        p.fill_drafts(rng)
        clean = (p.latent.copy(), p.rope.copy())
        words = tree_words(rng, p.toks, "tree")
        bads = [(0, 4), (0, 7), (1, 0)]
        for k, (b, j) in enumerate(bads):
            r = p.rows(b)[p.lens[b] + j]
            p.latent[r, [3, 300][k % 2]] = bad
            if k == 1:
                p.rope[r] = bad
                p.latent[r] = bad
        p.up()
        x = tree_inputs(ctx, rng, p, H)
        got = run_tree(ctx, p, x, words, H, 0.0722)
        p.latent, p.rope = clean
        f = lambda a: W.bf16_to_f32(a).astype(np.float64)  # noqa: E731
        want, lim = tree_oracle(p, words, *(f(a) for a in x), 0.0722)
        for b in range(2):
            for i in range(p.toks[b]):
                t = int(p.cu[b]) + i
                if any(bb == b and (int(words[t]) >> j) & 1 for bb, j in bads):
                    assert np.isnan(got[t]).all(), (bad, b, i)
                else:
                    assert (np.abs(got[t] - want[t]) <= lim[t]).all(), (bad, b, i)


def test_tree_is_deterministic_and_fresh(ctx):
    """The same bits whatever the workspace held and whatever ran before."""
    rng = np.random.default_rng(11)
    p, x, words, got = check_tree(ctx, rng, [900, 33, 4000], [8, 1, 5], 32, 24, "tree", pad=1)
    n = ctx.mla_tree_attend_workspace(3, p.T, 24)
    ws = ctx.empty((n,), np.uint8) if n else None
    for _ in range(3):
        again = run_tree(ctx, p, x, words, 24, 0.0722, ws=ws)
        tot = int(p.cu[-1])
        assert (again[:tot].view(np.uint32) == got[:tot].view(np.uint32)).all()


def test_tree_reports_bad_tables(ctx):
    rng = np.random.default_rng(12)
    for what, text in (("page", "outside the cache"), ("len", "negative length"),
                       ("table", "page table"), ("cu", "cu_tokens"), ("many", "more new tokens")):
        p = Paged(ctx, rng, [20, 30, 10], [2, 3, 70 if what == "many" else 3], 16)
        p.fill_drafts(rng)
        good = [0] if what in ("many", "cu") else [0, 2]
        x = tree_inputs(ctx, rng, p, 4)
        words = tree_words(rng, [min(t, 64) for t in p.toks], "chain")
        words = np.concatenate([words, np.zeros(p.T - len(words), np.uint64)])
        f = lambda a: W.bf16_to_f32(a).astype(np.float64)  # noqa: E731
        keep = (p.toks, p.lens, p.cu)
        p.toks = [t if b in good else 0 for b, t in enumerate(p.toks)]
        want, lim = tree_oracle(p, words, *(f(a) for a in x), 0.0722)
        p.toks = keep[0]
        if what == "page":
            p.table[1, 0] = -1
        if what == "len":
            p.lens = [20, -5, 10]
        if what == "table":
            p.lens = [20, p.width * 16, 10]
        if what == "cu":
            p.cu = np.array([0, 2, 2000000000, -4], np.int32)
            p.cu[3] = p.T
        p.up()
        dx = [ctx.upload(a) for a in x]
        dm = ctx.upload(words)
        out = ctx.empty((p.T, 4, 128), np.float32)
        out.zero()
        n = ctx.mla_tree_attend_workspace(3, p.T, 4)
        ws = ctx.empty((max(n, 1),), np.uint8)
        ctx.mla_tree_attend(out, dx[0], dx[1], p.cache, p.batch, dx[2], dx[3], 4, 0.0722, ws, n,
                            tree_mask=dm)
        with pytest.raises(k3cuda.K3CudaError, match=text) as e:
            ctx.sync()
        assert e.value.code == k3cuda.ERR_ARG
        got = out.numpy()
        for b in good:
            t = slice(int(keep[2][b]), int(keep[2][b + 1]))
            assert (np.abs(got[t] - want[t]) <= lim[t]).all(), (what, b)


@pytest.mark.parametrize("cu,good", OUT_OF_ORDER)
def test_tree_offsets_out_of_order(ctx, cu, good):
    """The sequences that the append takes, and no others."""
    rng = np.random.default_rng(15)
    p = out_of_order(ctx, rng, cu, good)
    x = tree_inputs(ctx, rng, p, 4)
    n = ctx.mla_tree_attend_workspace(3, 8, 4)
    out, ws = ctx.empty((8, 4, 128), np.float32), ctx.empty((n,), np.uint8)
    out.fill(0x4B)
    ws.fill(0xFF)
    dx = [ctx.upload(a) for a in x]
    ctx.mla_tree_attend(out, dx[0], dx[1], p.cache, p.batch, dx[2], dx[3], 4, 0.0722, ws, n)
    reports(ctx, "cu_tokens")
    got, told = out.numpy(), np.zeros(8, bool)
    for b in range(good):
        told[cu[b]:cu[b + 1]] = True
    words = np.zeros(8, np.uint64)
    for b in range(good):
        words[cu[b]:cu[b + 1]] = tree_words(rng, [p.toks[b]], "chain")
    p.toks = [t if b < good else 0 for b, t in enumerate(p.toks)]
    f = lambda a: W.bf16_to_f32(a).astype(np.float64)  # noqa: E731
    want, lim = tree_oracle(p, words, *(f(a) for a in x), 0.0722)
    assert (np.abs(got[told] - want[told]) <= lim[told]).all()
    assert (got[~told].view(np.uint32) == 0x4B4B4B4B).all()


def test_refused_sequences_stay_as_they_were(ctx):
    """A sequence that another rule leaves out: its cache rows, queries and outputs."""
    rng = np.random.default_rng(16)
    for what, lens in (("length", [20, -1, 10]), ("table", [20, 1 << 20, 10]), ("drafts", [20, 30, 10])):
        toks = [2, 65 if what == "drafts" else 3, 3]
        p = Paged(ctx, rng, [20, 30, 10], toks, 16)
        p.fill_drafts(rng)
        p.lens = lens
        p.up()
        bad = slice(2, 2 + toks[1])
        x = tree_inputs(ctx, rng, p, 4)
        dx = [ctx.upload(a) for a in x]
        n = ctx.mla_tree_attend_workspace(3, p.T, 4)
        out, ws = ctx.empty((p.T, 4, 128), np.float32), ctx.empty((n,), np.uint8)
        out.fill(0x4B)
        ctx.mla_tree_attend(out, dx[0], dx[1], p.cache, p.batch, dx[2], dx[3], 4, 0.0722, ws, n)
        reports(ctx, {"length": "negative", "table": "page table", "drafts": "more new"}[what])
        got = out.numpy()
        assert (got[bad].view(np.uint32) == 0x4B4B4B4B).all(), what
        assert (np.delete(got, np.arange(p.T)[bad], 0).view(np.uint32) != 0x4B4B4B4B).all(), what
        if what == "drafts":
            continue   # the append takes any number of tokens
        q = rng.standard_normal((p.T, 4, 192)).astype(np.float32)
        dq, dct = ctx.upload(q), ctx.upload(rng.standard_normal((p.T, 576)).astype(np.float32))
        dw = ctx.upload(np.ones(512, np.float32))
        qn, qr = (ctx.upload(np.full((p.T, 4, m), 0x1234, np.uint16)) for m in (128, 64))
        ctx.mla_paged_append(p.cache, p.batch, dct, dw, 1e-6, q=dq, q_nope=qn, q_rope=qr, H=4)
        reports(ctx, {"length": "negative", "table": "page table", "drafts": "more new"}[what])
        assert (qn.numpy()[bad] == 0x1234).all() and (qr.numpy()[bad] == 0x1234).all(), what
        p.lens = [20, 30, 10]
        rest = np.ones(len(p.latent), bool)
        for b in (0, 2):
            rest[p.rows(b)[p.lens[b]:]] = False
        assert (p.d[0].numpy()[rest] == p.latent[rest]).all(), what
        assert (p.d[1].numpy()[rest] == p.rope[rest]).all(), what


# ------------------------------------------------------------------------ log probabilities
def lp_oracle(x, tokens, K):
    T, V = x.shape
    x = x.astype(np.float64)
    lp = np.full(tokens.shape, -np.inf)
    ent, ids, tlp = np.full(T, np.nan), np.full((T, K), -1), np.full((T, K), np.nan)
    for r in range(T):
        m = x[r].max()
        if not np.isfinite(m):       # NaN, +inf, or nothing but -inf
            lp[r] = np.nan
            continue
        with np.errstate(over="ignore"):
            e = np.exp(x[r] - m)
        s = e.sum()
        d = np.where(e > 0, x[r] - m, 0)
        ent[r] = np.log(s) - (e * d).sum() / s
        ok = (tokens[r] >= 0) & (tokens[r] < V)
        lp[r, ok] = x[r, tokens[r, ok]] - m - np.log(s)
        order = np.lexsort((np.arange(V), -x[r]))[:K]
        order = order[x[r, order] > -np.inf]
        ids[r, :len(order)] = order
        tlp[r] = -np.inf
        tlp[r, :len(order)] = x[r, order] - m - np.log(s)
    return lp, ent, ids, tlp


def run_lp(ctx, x, tokens, K, bf16, stride=None, shift=0, entropy=True):
    """x [T][V] fp32 (bf16-representable for bf16); rows `stride` apart, `shift` elements in."""
    T, V = x.shape
    stride = stride or V
    dt = np.uint16 if bf16 else np.float32
    buf = np.full(shift + max(T, 1) * stride, 0x7F80 if bf16 else np.inf, dt)  # +inf between rows
    for r in range(T):
        buf[shift + r * stride: shift + r * stride + V] = W.f32_to_bf16(x[r]) if bf16 else x[r]
    d = ctx.upload(buf)
    G = tokens.shape[1]
    dtok = ctx.upload(tokens.astype(np.int32)) if tokens.size else None
    lp, ent = ctx.empty((max(T * G, 1),), np.float32), ctx.empty((max(T, 1),), np.float32)
    ids, tlp = ctx.empty((max(T * K, 1),), np.int32), ctx.empty((max(T * K, 1),), np.float32)
    n = ctx.token_logprobs_workspace(T, V, K)
    ws = ctx.empty((max(n, 1),), np.uint8)
    ws.fill(0xFF)
    ctx.token_logprobs(d.ptr + shift * dt().itemsize, T, V, dtok, G, lp if G else None, ws, n,
                       entropy=ent if entropy else None, K=K, top_ids=ids if K else None,
                       top_logprobs=tlp if K else None, io_dtype=k3cuda.BF16 if bf16 else k3cuda.F32,
                       row_stride=stride)
    ctx.sync()
    return (lp.numpy()[:T * G].reshape(T, G), ent.numpy()[:T], ids.numpy()[:T * K].reshape(T, K),
            tlp.numpy()[:T * K].reshape(T, K))


def check_lp(ctx, x, tokens, K, bf16, **kw):
    """A thread sums up to n = V/256 + 40 terms in a row, the joins add 20 more; each term carries
    the rounding of x - m, of its scaling to log2 units (both relative to the exponent, below
    90 where a term counts) and 2^-21 of ex2. A log probability adds the roundings of x - m and
    the difference."""
    lp, ent, ids, tlp = run_lp(ctx, x, tokens, K, bf16, **kw)
    with np.errstate(invalid="ignore"):
        w_lp, w_ent, w_ids, w_tlp = lp_oracle(x, tokens, K)
    rel = (x.shape[1] / 256 + 60 + 3 * 90) * F4 + 2.0 ** -21

    def same(got, want, off):
        assert (np.isnan(got) == np.isnan(want)).all()
        inf = np.isinf(want)
        assert (got[inf] == want[inf]).all()
        f = np.isfinite(want)
        assert (np.abs(got[f] - want[f]) <= np.broadcast_to(off, want.shape)[f]).all(), \
            np.abs(got[f] - want[f]).max()
    with np.errstate(invalid="ignore"):
        same(lp, w_lp, rel + 6 * F4 * np.abs(w_lp))
        same(tlp, w_tlp, rel + 6 * F4 * np.abs(w_tlp))
        # t/s: both sums off by rel, |t/s| <= entropy + log s <= 2 log V
        same(ent, w_ent, rel * (1 + 4 * np.log(x.shape[1] + 1)) + 4 * F4)
    assert (ids == w_ids).all()
    return lp, ent, ids, tlp


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("T,V,G,K", [(1, 1, 1, 1), (2, 2, 1, 4), (3, 31, 2, 32), (5, 1000, 3, 20),
                                     (4, 1001, 1, 8), (3, 4097, 1, 5), (7, 50257, 4, 5),
                                     (1, 163840, 1, 8), (2, 131072, 0, 32), (300, 777, 1, 0),
                                     (1300, 2049, 2, 9), (160, 32001, 1, 17)])
def test_logprobs(ctx, bf16, T, V, G, K):
    rng = np.random.default_rng([T, V, K])
    x = rng.standard_normal((T, V)).astype(np.float32) * 2.5
    if V > 100:
        x[:, rng.integers(0, V, 3)] += 9
        x[::3, V // 3: V // 2] = -np.inf
    if bf16:
        x = W.round_bf16(x)
    tokens = rng.integers(0, V, (T, G))
    check_lp(ctx, x, tokens, K, bf16)


@pytest.mark.parametrize("bf16", [False, True])
def test_logprobs_rows_at_any_alignment(ctx, bf16):
    rng = np.random.default_rng(3)
    for V, stride, shift in ((513, 517, 1), (9, 9, 3), (4001, 4005, 7), (70001, 70003, 5)):
        x = rng.standard_normal((6, V)).astype(np.float32)
        x = W.round_bf16(x) if bf16 else x
        check_lp(ctx, x, rng.integers(0, V, (6, 2)), 6, bf16, stride=stride, shift=shift)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("V", [40, 3000, 163841])
def test_logprobs_odd_rows(ctx, bf16, V):
    """Rows without a distribution, with fewer tokens than places, with equal logits (more than
    the ranking takes at once), with zeros of both signs, large logits, tokens out of range."""
    rng = np.random.default_rng(V)
    x = rng.standard_normal((12, V)).astype(np.float32)
    x[0] = -np.inf
    x[1, V // 2] = np.nan
    x[2, V - 1] = np.inf
    x[3] = -np.inf
    x[3, [V - 1, 3, V // 2]] = [1.0, 2.0, 1.0]
    x[4] = 0.25
    x[5] = np.where(np.arange(V) % 3 == 0, 0.0, -0.0)
    x[6] = 1000 + 8 * rng.integers(0, 3, V)
    x[7] = np.arange(V) % 7
    x[8] = -np.inf
    x[8, 5] = -3.0
    x[9] = 60000 * np.sign(x[9])
    x[10, :3] = np.nan
    x[11] = np.sort(x[11])
    x = W.round_bf16(x) if bf16 else x
    x[1, V // 2] = x[10, 0] = x[10, 1] = x[10, 2] = np.nan
    tokens = np.stack([rng.integers(0, V, 12), np.full(12, -1), np.full(12, V),
                       np.full(12, 2 ** 31 - 1), np.full(12, 5)], 1)
    lp, ent, ids, tlp = check_lp(ctx, x, tokens, 30, bf16)
    assert ids[5, :5].tolist() == [0, 1, 2, 3, 4]
    assert ids[3, :4].tolist() == [3, V // 2, V - 1, -1]
    assert lp[8, 4] == 0 and ent[8] == 0
    again = run_lp(ctx, x, tokens, 30, bf16, entropy=False)
    assert (again[2] == ids).all() and np.array_equal(again[0], lp, equal_nan=True)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("T,V", [(1, 163840), (620, 20000), (100, 30001)])
def test_logprobs_few_tokens_allowed(ctx, bf16, T, V):
    """All but a few tokens forbidden: warps, blocks and segments without one, or with one thread's."""
    rng = np.random.default_rng([T, V])
    x = np.full((T, V), -np.inf, np.float32)
    for r in range(T):
        n = [1, 5, 300, 4000][r % 4 if T > 1 else 2]
        at = rng.integers(0, V, n) if r % 8 < 4 else (17 + 256 * np.arange(n)) % V
        x[r, at] = rng.standard_normal(n) * 3
    x = W.round_bf16(x) if bf16 else x
    check_lp(ctx, x, rng.integers(0, V, (T, 2)), 32 if T == 1 else 8, bf16)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("T,V", [(2, 163840), (300, 50000)])
def test_logprobs_likeliest_in_few_threads(ctx, bf16, T, V):
    """Likely tokens that a few threads of a block read (they lie a fixed stride apart), all the
    others far below; distinct and in classes of equal ones. Of 300 rows with 24 in 1024 more reach
    the bound than are ranked at once."""
    rng = np.random.default_rng([T, V])
    for stride, some, K in ((4096, 40, 20), (1024, 24, 32), (8192, 64, 9), (2048, 16, 30)):
        x = rng.standard_normal((T, V)).astype(np.float32)
        x[:, np.arange(V) % stride < some] += 20
        x[1::2] = np.round(x[1::2])
        x = W.round_bf16(x) if bf16 else x
        check_lp(ctx, x, rng.integers(0, V, (T, 1)), K, bf16)


def lp_time(ctx, x, K):
    """Shortest of several device times of a call, in ms, with cold caches."""
    T, V = x.shape
    d, n = ctx.upload(x), ctx.token_logprobs_workspace(T, V, K)
    ws, lp = ctx.empty((max(n, 1),), np.uint8), ctx.empty((T, 1), np.float32)
    dtok, ids = ctx.upload(np.zeros((T, 1), np.int32)), ctx.empty((T, K), np.int32)
    tlp, best = ctx.empty((T, K), np.float32), 1e9
    for k in range(6):
        ctx.flush_l2()
        ctx.record(0)
        ctx.token_logprobs(d, T, V, dtok, 1, lp, ws, n, K=K, top_ids=ids, top_logprobs=tlp)
        ctx.record(1)
        ctx.sync()
        best = min(best, ctx.elapsed_ms(0, 1)) if k > 1 else best
    return best


@pytest.mark.parametrize("T,V", [(600, 163840), (7, 163840), (64, 50257)])
def test_logprobs_of_logits_with_a_large_offset(ctx, T, V):
    """Distinct fp32 logits around -1030, 1030 and 2^20: what a row's softmax does not see does not
    change its ids, and costs no further passes over the row; nor do equal logits."""
    rng = np.random.default_rng([T, V])
    z = rng.standard_normal((T, V)).astype(np.float32) * 2.5
    for off in (-1030.0, 1030.0, 2.0 ** 20):
        x = z + np.float32(off)
        if T < 100:
            check_lp(ctx, x, rng.integers(0, V, (T, 2)), 20, False)
        else:
            ids = run_lp(ctx, x, rng.integers(0, V, (T, 1)), 20, False)[2]
            order = np.argsort(-x[::60], axis=1, kind="stable")[:, :20]
            assert (ids[::60] == order).all()
            if off < 2.0 ** 19:   # at 2^20 thousands of logits are equal
                assert lp_time(ctx, x, 20) < 2 * lp_time(ctx, z, 20)


def test_logprobs_nothing_to_do(ctx):
    run_lp(ctx, np.zeros((0, 50), np.float32), np.zeros((0, 1), np.int64), 3, False)
    run_lp(ctx, np.zeros((3, 50), np.float32), np.zeros((3, 0), np.int64), 0, False)


# --------------------------------------------------------------------------------- together
def verify_step(ctx, p, data, H, V, words, bufs):
    """One verification step: append, attend, vocabulary projection, log probabilities."""
    ctx.mla_paged_append(p.cache, p.batch, data["ct"], data["w"], 1e-6, q=data["q"],
                         q_nope=bufs["qn"], q_rope=bufs["qr"], H=H, positions=data["pos"],
                         inv_freq=data["inv"])
    ctx.mla_tree_attend(bufs["out"], bufs["qn"], bufs["qr"], p.cache, p.batch, data["uk"],
                        data["uv"], H, 0.0722, bufs["ws"], bufs["nws"], tree_mask=words)
    ctx.matmul(bufs["logits"], bufs["out"], data["head"], k3cuda.F32, H * 128, V, p.T)
    ctx.token_logprobs(bufs["logits"], p.T, V, data["tok"], 1, bufs["lp"], bufs["ws2"],
                       bufs["nws2"], entropy=bufs["ent"], K=4, top_ids=bufs["ids"],
                       top_logprobs=bufs["tlp"])


def step_data(ctx, rng, p, H, V):
    g = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
    b = W.f32_to_bf16
    host = dict(ct=g(p.T, 576), w=np.ones(512, np.float32), q=g(p.T, H, 192),
                pos=rng.integers(0, 10000, p.T).astype(np.int32),
                inv=(10000.0 ** (-np.arange(32) / 32)).astype(np.float32),
                uk=b(g(H, 128, 512) * 0.04), uv=b(g(H, 128, 512) * 0.04), head=g(V, H * 128),
                tok=rng.integers(0, V, (p.T, 1)).astype(np.int32))
    dev = {k: ctx.upload(v) for k, v in host.items()}
    n, n2 = ctx.mla_tree_attend_workspace(len(p.lens), p.T, H), ctx.token_logprobs_workspace(
        p.T, V, 4)
    bufs = dict(qn=ctx.empty((p.T, H, 128), np.uint16), qr=ctx.empty((p.T, H, 64), np.uint16),
                out=ctx.empty((p.T, H, 128), np.float32), nws=n, ws=ctx.empty((max(n, 1),), np.uint8),
                logits=ctx.empty((p.T, V), np.float32), nws2=n2,
                ws2=ctx.empty((max(n2, 1),), np.uint8), lp=ctx.empty((p.T, 1), np.float32),
                ent=ctx.empty((p.T,), np.float32), ids=ctx.empty((p.T, 4), np.int32),
                tlp=ctx.empty((p.T, 4), np.float32))
    return host, dev, bufs


def test_a_verification_step(ctx):
    """The three operators as a serving step runs them, twice, the second step over the rows that
    the first one appended; each result against its own 64-bit form on the step's own inputs."""
    rng = np.random.default_rng(20)
    H, V = 8, 1003
    p = Paged(ctx, rng, [50, 0, 129], [6, 3, 7], 16)
    host, dev, bufs = step_data(ctx, rng, p, H, V)
    f = lambda a: W.bf16_to_f32(a).astype(np.float64)  # noqa: E731
    words = tree_words(rng, p.toks, "tree")
    dw = ctx.upload(words)
    for step in range(2):
        verify_step(ctx, p, dev, H, V, dw, bufs)
        ctx.sync()
        p.latent, p.rope = p.d[0].numpy(), p.d[1].numpy()
        want, lim = tree_oracle(p, words, f(bufs["qn"].numpy()), f(bufs["qr"].numpy()),
                                f(host["uk"]), f(host["uv"]), 0.0722)
        out = bufs["out"].numpy()
        assert (np.abs(out - want) <= lim).all()
        logits = bufs["logits"].numpy()
        w_lp, w_ent, w_ids, w_tlp = lp_oracle(logits, host["tok"], 4)
        assert (bufs["ids"].numpy() == w_ids).all()
        off = 1e-5 * (1 + np.abs(w_lp))   # sums of 1003 terms in fp32
        assert (np.abs(bufs["lp"].numpy() - w_lp) <= off).all()
        assert (np.abs(bufs["tlp"].numpy() - w_tlp) <= 1e-5 * (1 + np.abs(w_tlp))).all()
        if step == 0:
            # two drafts of each sequence are accepted (rows stay where they are)
            p.lens = [ln + 2 for ln in p.lens]
            p.toks = [5, 1, 6]
            p.cu = np.concatenate([[0], np.cumsum(p.toks)]).astype(np.int32)
            words = tree_words(rng, p.toks, "tree")
            dw = ctx.upload(np.concatenate([words, np.zeros(p.T, np.uint64)]))
            words = np.concatenate([words, np.zeros(p.T - len(words), np.uint64)])
            p.T = int(p.cu[-1])
            p.up()
            host, dev, bufs = step_data(ctx, rng, p, H, V)


class Graph:
    """What the library issues on a context's stream, captured and replayed through the CUDA
    runtime that it is linked against."""

    def __init__(self, ctx, fn):
        self.rt = C.CDLL("libcudart.so.12")
        self.stream = C.c_void_p(k3cuda.lib().k3cuda_stream(ctx.h))
        graph, self.exe = C.c_void_p(), C.c_void_p()
        assert self.rt.cudaStreamBeginCapture(self.stream, 1) == 0   # this thread's calls
        try:
            fn()
        finally:
            rc = self.rt.cudaStreamEndCapture(self.stream, C.byref(graph))
        assert rc == 0
        assert self.rt.cudaGraphInstantiate(C.byref(self.exe), graph, C.c_ulonglong(0)) == 0
        assert self.rt.cudaGraphDestroy(graph) == 0

    def replay(self):
        assert self.rt.cudaGraphLaunch(self.exe, self.stream) == 0

    def close(self):
        assert self.rt.cudaGraphExecDestroy(self.exe) == 0


def test_captured_step_replays_with_new_lengths(ctx):
    """A captured step reads lengths, offsets and pages when it is replayed; two captured steps
    with a workspace each do not disturb one another."""
    rng = np.random.default_rng(21)
    H, V = 8, 1003
    parts = []
    for k in range(2):
        p = Paged(ctx, rng, [200, 90], [4, 4], 16)
        host, dev, bufs = step_data(ctx, rng, p, H, V)
        dw = ctx.upload(tree_words(rng, p.toks, "chain"))
        verify_step(ctx, p, dev, H, V, dw, bufs)   # warm: attributes are set outside the capture
        ctx.sync()
        parts.append((p, dev, bufs, dw,
                      Graph(ctx, lambda: verify_step(ctx, p, dev, H, V, dw, bufs))))
    names = ("out", "lp", "ent", "ids", "tlp")
    for lens, toks in (([200, 90], [4, 4]), ([33, 0], [1, 7]), ([0, 150], [8, 0])):
        want = []
        for p, dev, bufs, dw, g in parts:
            cu = np.concatenate([[0], np.cumsum(toks)]).astype(np.int32)
            p.d[3].copy_from(np.asarray(lens, np.int32))
            p.d[4].copy_from(cu)
            for n in names:
                bufs[n].zero()
            verify_step(ctx, p, dev, H, V, dw, bufs)
            ctx.sync()
            want.append([bufs[n].numpy() for n in names])
            for n in names:
                bufs[n].zero()
        ctx.sync()
        for _ in range(2):
            for part in parts:
                part[4].replay()
        ctx.sync()
        for (p, dev, bufs, dw, g), w in zip(parts, want):
            for n, a in zip(names, w):
                assert np.array_equal(bufs[n].numpy(), a, equal_nan=True), n
    for part in parts:
        part[4].close()


def test_buffers_freed_while_a_step_is_captured(ctx):
    """Frees of device and page-locked memory, as a garbage collector may make them at any time,
    do not end a capture."""
    rng = np.random.default_rng(23)
    H, V = 4, 501
    p = Paged(ctx, rng, [60], [3], 16)
    host, dev, bufs = step_data(ctx, rng, p, H, V)
    dw = ctx.upload(tree_words(rng, p.toks, "chain"))
    verify_step(ctx, p, dev, H, V, dw, bufs)
    ctx.sync()
    want = {n: bufs[n].numpy() for n in ("out", "lp", "ids")}
    spare, pinned = [ctx.empty((1 << 20,), np.uint8) for _ in range(2)], ctx.host_alloc(4096)

    def step():
        spare[0].free()
        verify_step(ctx, p, dev, H, V, dw, bufs)
        ctx.host_free(pinned)
        spare[1].free()

    g = Graph(ctx, step)
    for n in want:
        bufs[n].zero()
    g.replay()
    ctx.sync()
    for n, a in want.items():
        assert np.array_equal(bufs[n].numpy(), a), n
    g.close()


def test_two_contexts_at_once(ctx):
    """Two contexts (streams) run steps on caches and workspaces of their own at the same time."""
    rng = np.random.default_rng(22)
    H, V = 16, 2001
    with k3cuda.Context(ctx.device) as other:
        parts = []
        for c in (ctx, other):
            p = Paged(c, rng, [3000, 1500], [8, 5], 64)
            host, dev, bufs = step_data(c, rng, p, H, V)
            dw = c.upload(tree_words(rng, p.toks, "tree"))
            parts.append((c, p, dev, bufs, dw))
        for c, p, dev, bufs, dw in parts:
            verify_step(c, p, dev, H, V, dw, bufs)
            c.sync()
        want = [[q[3][n].numpy() for n in ("out", "lp", "ids")] for q in parts]
        for _ in range(10):
            for c, p, dev, bufs, dw in parts:
                verify_step(c, p, dev, H, V, dw, bufs)
        for q, w in zip(parts, want):
            q[0].sync()
            for n, a in zip(("out", "lp", "ids"), w):
                assert np.array_equal(q[3][n].numpy(), a), n
        del parts, q, p, dev, bufs, dw
