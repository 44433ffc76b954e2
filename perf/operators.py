"""Cases of the draft-verification operators: the step that checks drafted tokens against a model.

A serving step with speculative decoding makes three calls beyond the projections:

  append    the drafted tokens' queries and cache rows: the latent normalised, the rope slots of
            queries and keys rotated, the rows written into a paged latent cache
  attend    absorbed latent attention of every drafted token over its sequence's cached rows and
            its own ancestors in the tree of drafts
  logprobs  log probabilities of given tokens, the entropy and the top alternatives of each row
            of logits

``listed`` and ``draw`` give cases, ``prepare`` makes what a serving program has in hand before
the call, ``run`` makes one pass: with ``own`` false in elementary fp32 torch operations, with
``own`` true through the library. ``exact`` states the same results in 64 bits.
"""
import math
import os
import random
import sys

import torch

own = False

DN, DR, DL, DV = 128, 64, 512, 128      # head geometry of the latent attention
EPS = 1e-6
THETA = 50000.0                         # rotation base of the rope slot
POSITIONS = 1 << 20                     # positions an append may start from (long contexts)
DEV = "cuda"


# ------------------------------------------------------------------------------ cases
def listed():
    return [
        # one new token for each of 64 running requests: the smallest append, latency counts
        dict(name="append decode 64x1", op="append", B=64, n=1, ragged=False, H=16, page=64,
             ctx=1024, io="f32", style="half", lens=1),
        # drafts of odd lengths for 13 requests on short pages, bf16 projections
        dict(name="append drafts 13x26", op="append", B=13, n=26, ragged=True, H=96, page=16,
             ctx=2000, io="bf16", style="interleaved", lens=2),
        # prompts of three requests, all heads on one GPU: the largest append
        dict(name="append prompt 3x4096", op="append", B=3, n=4096, ragged=True, H=128, page=64,
             ctx=512, io="f32", style="half", lens=3),
        # one token after a short prompt, the heads of one of eight ranks: the smallest attention
        dict(name="attend 1x1 ctx 509 H 16", op="attend", B=1, n=1, ragged=False, H=16, page=64,
             ctx=509, spread=False, lens=4),
        # plain decoding of a full batch, no drafts: 64 sequences of 8192 positions, 128 heads
        dict(name="attend 64x1 ctx 8192 H 128", op="attend", B=64, n=1, ragged=False, H=128,
             page=64, ctx=8192, spread=False, lens=5),
        # trees of up to 16 drafts, one of eight ranks, contexts of every length
        dict(name="attend 64x16 ctx 8192 H 16", op="attend", B=64, n=16, ragged=True, H=16,
             page=32, ctx=8192, spread=True, lens=6),
        # trees of up to 13 drafts with all 128 heads on one GPU: the largest attention
        dict(name="attend 48x13 ctx 8192 H 128", op="attend", B=48, n=13, ragged=True, H=128,
             page=64, ctx=8192, spread=True, lens=7),
        # one request with a long context and a tree of 26 drafts, 12 heads of one rank
        dict(name="attend 1x26 ctx 131071 H 12", op="attend", B=1, n=26, ragged=False, H=12,
             page=128, ctx=131071, spread=False, lens=8),
        # one row of logits: the smallest call
        dict(name="logprobs 1x163840 bf16", op="logprobs", T=1, V=163840, io="bf16", G=1, K=8),
        # the drafts of 13 requests, an odd vocabulary, several children to score at each node
        dict(name="logprobs 209x50257 f32", op="logprobs", T=209, V=50257, io="f32", G=4, K=5),
        # a batch of drafts over a large vocabulary
        dict(name="logprobs 512x163840 f32", op="logprobs", T=512, V=163840, io="f32", G=2, K=20),
        # the log probabilities of a whole prompt: the largest call
        dict(name="logprobs 2048x163840 bf16", op="logprobs", T=2048, V=163840, io="bf16", G=1,
             K=1),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "logprobs"])
    if op == "append":
        B = _log(rng, 1, 96)
        n = _log(rng, 1, 4096 // B)
        return dict(op=op, B=B, n=n, ragged=rng.random() < 0.7, H=rng.choice([12, 16, 96, 128]),
                    page=rng.choice([16, 32, 64, 128]), ctx=_log(rng, 1, 4096),
                    io=rng.choice(["f32", "bf16"]), style=rng.choice(["half", "interleaved"]),
                    lens=rng.randrange(1 << 30))
    if op == "attend":
        H = rng.choice([8, 12, 16, 32, 96, 128])
        n = _log(rng, 1, 64)
        B = _log(rng, 1, min(64, 1024 // n))
        # scores below those of a full batch's decoding, and a cache of 1 M positions at most
        ctx = min((48 * 128 * 8192) // (B * n * H), (1 << 20) // B, 131072)
        return dict(op=op, B=B, n=n, ragged=rng.random() < 0.7, H=H,
                    page=rng.choice([16, 32, 64, 128]), ctx=_log(rng, 1, max(2, ctx)),
                    spread=rng.random() < 0.6, lens=rng.randrange(1 << 30))
    V, io = _log(rng, 1000, 200000), rng.choice(["f32", "bf16"])
    most = 2048 * 163840 // V // (2 if io == "f32" else 1)
    return dict(op=op, T=_log(rng, 1, min(4096, most)), V=V, io=io, G=rng.randint(1, 6),
                K=rng.randint(0, 20))


def _lengths(case):
    """(cached rows, drafted tokens) of every sequence: part of the case, not of the seed."""
    r = random.Random(case["lens"])
    lens, toks = [], []
    for _ in range(case["B"]):
        spread = case.get("spread", True)
        lens.append(r.randint(0, case["ctx"]) if spread else case["ctx"])
        toks.append(r.randint(0, case["n"]) if case["ragged"] else case["n"])
    if sum(toks) == 0:
        toks[0] = case["n"]
    if case.get("spread", True):
        lens[-1] = case["ctx"]
    return lens, toks


def work(case):
    if case["op"] == "logprobs":
        T, V, G, K = case["T"], case["V"], case["G"], case["K"]
        size = 4 if case["io"] == "f32" else 2
        # per logit: a maximum, an exponential and two sums
        return {"bytes": T * (V * size + 8 * G + 4 + 8 * K), "flops": 5 * T * V}
    lens, toks = _lengths(case)
    H, T = case["H"], sum(toks)
    if case["op"] == "append":
        size = 4 if case["io"] == "f32" else 2
        return {"bytes": T * ((DL + DR) * (size + 2) + H * (DN + DR) * (size + 2)) + DL * 4,
                "flops": T * (4 * DL + 3 * DR + 3 * H * DR)}
    rows = sum(ln + t for ln, t in zip(lens, toks) if t)
    pairs = sum((ln + 1) * t for ln, t in zip(lens, toks))   # every token sees itself too
    absorb = 2 * T * H * DL * (DN + DV)
    return {"bytes": rows * (DL + DR) * 2 + T * H * (DN + DR + DV) * 2 + 2 * H * 128 * DL * 2,
            "flops": 2 * pairs * H * (2 * DL + DR) + absorb}


# ------------------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _normal(g, shape, std=1.0, dtype=torch.bfloat16):
    return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32).mul_(std).to(dtype)


def _prepare_logprobs(case, seed):
    g = _gen(seed)
    T, V, G, K = case["T"], case["V"], case["G"], case["K"]
    dt = torch.float32 if case["io"] == "f32" else torch.bfloat16
    logits = _normal(g, (T, V), 2.5, dt)
    # a few likely tokens in every row, a stretch that a grammar forbids in every third
    first = torch.randint(0, V, (T, 1), generator=g, device=DEV)
    likely = (first + torch.arange(8, device=DEV) * (V // 8)) % V
    logits.scatter_add_(1, likely, _normal(g, (T, 8), 3.0, torch.float32).abs_().add_(6).to(dt))
    if V > 64:
        logits[::3, V // 3: V // 2] = float("-inf")
    given = torch.randint(0, V, (T, G), generator=g, device=DEV, dtype=torch.int32)
    given[:, 0] = likely[:, 0].to(torch.int32)
    new = lambda shape, dt: torch.empty(shape, device=DEV, dtype=dt)  # noqa: E731
    return dict(case=case, logits=logits, given=given,
                logprobs=new((T, G), torch.float32), entropy=new((T,), torch.float32),
                top_ids=new((T, K), torch.int32), top_logprobs=new((T, K), torch.float32))


def _tree_masks(seed, toks):
    """Visible drafts of each drafted token (bit j: draft j of its sequence): itself and its
    ancestors in a random tree, every node's parent an earlier node or the last cached token."""
    r = random.Random(seed)
    words = []
    for n in toks:
        own_words = []
        for i in range(n):
            parent = r.randint(max(-1, i - 4), i - 1)
            own_words.append((own_words[parent] if parent >= 0 else 0) | (1 << i))
        words += own_words
    return [w - (1 << 64) if w >> 63 else w for w in words]


def prepare(case, seed):
    if case["op"] == "logprobs":
        return _prepare_logprobs(case, seed)
    g = _gen(seed)
    lens, toks = _lengths(case)
    B, H, page, T = case["B"], case["H"], case["page"], sum(toks)
    need = [(ln + t + page - 1) // page for ln, t in zip(lens, toks)]
    width = max(1, max(need))
    pool = sum(need) + 3
    # every sequence's pages lie scattered over the pool; entries behind its last one are unused
    perm = torch.randperm(pool, generator=g, device=DEV, dtype=torch.int32)
    table = torch.zeros((B, width), device=DEV, dtype=torch.int32)
    at = 0
    for b, k in enumerate(need):
        table[b, :k] = perm[at: at + k]
        at += k
    cu = [0]
    for t in toks:
        cu.append(cu[-1] + t)
    i32 = lambda v: torch.tensor(v, device=DEV, dtype=torch.int32)  # noqa: E731
    seq = torch.repeat_interleave(torch.arange(B, device=DEV), torch.tensor(toks, device=DEV))
    index = torch.arange(T, device=DEV) - i32(cu).long()[seq]     # place within its sequence
    s = dict(case=case, B=B, T=T, toks=toks, lens_host=lens, lens=i32(lens), cu=i32(cu),
             table=table, seq=seq, index=index,
             latent=_normal(g, (pool, page, DL), 0.5), rope=_normal(g, (pool, page, DR)))
    if case["op"] == "append":
        dt = torch.float32 if case["io"] == "f32" else torch.bfloat16
        base = torch.randint(0, POSITIONS, (B,), generator=g, device=DEV, dtype=torch.int32)
        s.update(ct=_normal(g, (T, DL + DR), 1.0, dt), q=_normal(g, (T, H, DN + DR), 1.0, dt),
                 weight=_normal(g, (DL,), 0.1, torch.float32).add_(1.0),
                 # as in a long conversation: the rotation's position need not be the row's place
                 positions=(base[seq] + index).to(torch.int32),
                 inv_freq=(THETA ** (-torch.arange(0, DR, 2, device=DEV, dtype=torch.float64)
                                     / DR)).float(),
                 q_nope=torch.empty((T, H, DN), device=DEV, dtype=torch.bfloat16),
                 q_rope=torch.empty((T, H, DR), device=DEV, dtype=torch.bfloat16))
        return s
    masks = _tree_masks(seed, toks)
    s.update(q_nope=_normal(g, (T, H, DN)), q_rope=_normal(g, (T, H, DR)),
             w_uk=_normal(g, (H, DN, DL), 0.02), w_uv=_normal(g, (H, DV, DL), 0.02),
             mask=torch.tensor(masks, device=DEV, dtype=torch.int64), nmax=max(toks),
             scale=1.0 / math.sqrt(DN + DR),
             out=torch.empty((T, H, DV), device=DEV, dtype=torch.bfloat16))
    return s


# ------------------------------------------------------------------------------ plain forms
def _rotate(x, cos, sin, style):
    if style == "half":
        a, b = x[..., : DR // 2], x[..., DR // 2:]
        return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)


def _plain_append(s):
    case = s["case"]
    ct, q = s["ct"].float(), s["q"].float()
    # angles of far positions lose their fraction in 32 bits
    angle = s["positions"].double()[:, None] * s["inv_freq"].double()
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    lat = ct[:, :DL]
    lat = lat / torch.sqrt((lat * lat).mean(-1, keepdim=True) + EPS) * s["weight"]
    key = _rotate(ct[:, DL:], cos, sin, case["style"])
    place = s["lens"][s["seq"]] + s["index"]
    row = s["table"][s["seq"], place // case["page"]].long() * case["page"] + place % case["page"]
    s["latent"].view(-1, DL)[row] = lat.to(torch.bfloat16)
    s["rope"].view(-1, DR)[row] = key.to(torch.bfloat16)
    s["q_nope"].copy_(q[..., :DN])
    s["q_rope"].copy_(_rotate(q[..., DN:], cos[:, None], sin[:, None], case["style"]))
    return s["latent"], s["rope"], s["q_nope"], s["q_rope"]


def _plain_attend(s):
    case = s["case"]
    B, n, H, page = s["B"], s["nmax"], case["H"], case["page"]
    cached, drafts = s["lens"].long(), (s["cu"][1:] - s["cu"][:-1]).long()
    longest = max(ln + t for ln, t in zip(s["lens_host"], s["toks"]))
    place = torch.arange(longest, device=DEV)
    row = s["table"][:, place // page].long() * page + place % page             # [B, longest]
    row = torch.where(place < (cached + drafts)[:, None], row, 0)
    lat, rope = s["latent"].view(-1, DL)[row].float(), s["rope"].view(-1, DR)[row].float()
    # queries in [B, n] boxes, absorbed: q W_UK
    box = s["seq"] * n + s["index"]
    qa = torch.einsum("thd,hdl->thl", s["q_nope"].float(), s["w_uk"].float())
    q_all = torch.cat([qa, s["q_rope"].float()], -1)
    q = torch.zeros((B * n, H, DL + DR), device=DEV).index_copy_(0, box, q_all)
    q = q.view(B, n * H, DL + DR)
    score = torch.bmm(q[..., :DL], lat.transpose(1, 2))
    score += torch.bmm(q[..., DL:], rope.transpose(1, 2))
    score = score.view(B, n, H, longest) * s["scale"]
    words = torch.zeros(B * n, device=DEV, dtype=torch.int64).index_copy_(0, box, s["mask"])
    draft = place[None] - cached[:, None]                                       # [B, longest]
    bit = (words.view(B, n, 1) >> draft.clamp(0, 63)[:, None]) & 1
    seen = (draft < 0)[:, None] | ((draft < drafts[:, None])[:, None] & (bit == 1))
    score = torch.where(seen[:, :, None], score, float("-inf"))
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(torch.isfinite(top), top, 0.0))
    total = p.sum(-1, keepdim=True)
    o = torch.bmm(p.view(B, n * H, longest), lat).view(B, n, H, DL)
    o = o / torch.where(total > 0, total, 1.0)
    o = o.view(B * n, H, DL)[box]
    s["out"].copy_(torch.einsum("thl,hvl->thv", o, s["w_uv"].float()))
    return s["out"]


def _plain_logprobs(s):
    x = s["logits"].float()
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(-1, keepdim=True)
    norm = top + torch.log(total)
    mean = (e * torch.where(torch.isinf(x), 0.0, x - top)).sum(-1) / total[:, 0]
    s["entropy"].copy_(torch.log(total[:, 0]) - mean)
    s["logprobs"].copy_(torch.gather(x, 1, s["given"].long()) - norm)
    if s["case"]["K"]:
        # equal logits in the order of their indices
        value, index = torch.sort(x, dim=1, descending=True, stable=True)
        index = torch.where(value == float("-inf"), -1, index)   # forbidden: no alternative
        s["top_ids"].copy_(index[:, : s["case"]["K"]])
        s["top_logprobs"].copy_(value[:, : s["case"]["K"]] - norm)
    return s["logprobs"], s["entropy"], s["top_ids"], s["top_logprobs"]


# ------------------------------------------------------------------------------ the library
_kept = {}   # the context and the workspace that a serving program keeps between calls


def _library():
    if "ctx" not in _kept:
        path = os.path.join(os.getcwd(), "kimi-k3-in-c_b200")
        if path not in sys.path:
            sys.path.insert(0, path)
        import k3cuda
        _kept["lib"] = k3cuda
        _kept["ctx"] = k3cuda.Context(torch.cuda.current_device())
    return _kept["lib"], _kept["ctx"]


def _workspace(nbytes):
    if "ws" not in _kept or _kept["ws"].numel() < nbytes:
        torch.cuda.synchronize()   # the old one may still be in use
        _kept["ws"] = torch.empty(max(nbytes, 1 << 20), device=DEV, dtype=torch.uint8)
    return _kept["ws"].data_ptr()


def _handles(s):
    """What a program keeps of a state between calls: the descriptors of cache and batch."""
    k3, _ = _library()
    if "cache" not in s:
        s["cache"] = k3.PagedCache(latent=s["latent"].data_ptr(), rope=s["rope"].data_ptr(),
                                   page_table=s["table"].data_ptr(),
                                   n_pages=s["latent"].shape[0], page_size=s["case"]["page"],
                                   max_pages=s["table"].shape[1])
        s["batch"] = k3.TokenBatch(ctx_lens=s["lens"].data_ptr(), cu_tokens=s["cu"].data_ptr(),
                                   B=s["B"], T=s["T"])
    return s["cache"], s["batch"]


def _own_append(s):
    k3, ctx = _library()
    cache, batch = _handles(s)
    case = s["case"]
    ctx.mla_paged_append(cache, batch, s["ct"].data_ptr(), s["weight"].data_ptr(), EPS,
                         q=s["q"].data_ptr(), q_nope=s["q_nope"].data_ptr(),
                         q_rope=s["q_rope"].data_ptr(), H=case["H"],
                         positions=s["positions"].data_ptr(), inv_freq=s["inv_freq"].data_ptr(),
                         rope_style=(k3.ROPE_HALF if case["style"] == "half"
                                     else k3.ROPE_INTERLEAVED),
                         io_dtype=k3.F32 if case["io"] == "f32" else k3.BF16)
    return s["latent"], s["rope"], s["q_nope"], s["q_rope"]


def _own_attend(s):
    k3, ctx = _library()
    cache, batch = _handles(s)
    H = s["case"]["H"]
    if "nws" not in s:
        s["nws"] = ctx.mla_tree_attend_workspace(s["B"], s["T"], H)
    ctx.mla_tree_attend(s["out"].data_ptr(), s["q_nope"].data_ptr(), s["q_rope"].data_ptr(),
                        cache, batch, s["w_uk"].data_ptr(), s["w_uv"].data_ptr(), H, s["scale"],
                        _workspace(s["nws"]), s["nws"], tree_mask=s["mask"].data_ptr(),
                        out_dtype=k3.BF16)
    return s["out"]


def _own_logprobs(s):
    k3, ctx = _library()
    case = s["case"]
    io = k3.F32 if case["io"] == "f32" else k3.BF16
    if "nws" not in s:
        s["nws"] = ctx.token_logprobs_workspace(case["T"], case["V"], case["K"])
    ctx.token_logprobs(s["logits"].data_ptr(), case["T"], case["V"], s["given"].data_ptr(),
                       case["G"], s["logprobs"].data_ptr(), _workspace(s["nws"]), s["nws"],
                       entropy=s["entropy"].data_ptr(), K=case["K"],
                       top_ids=s["top_ids"].data_ptr(), top_logprobs=s["top_logprobs"].data_ptr(),
                       io_dtype=io)
    return s["logprobs"], s["entropy"], s["top_ids"], s["top_logprobs"]


def run(state):
    op = state["case"]["op"]
    if own:
        return {"append": _own_append, "attend": _own_attend, "logprobs": _own_logprobs}[op](state)
    return {"append": _plain_append, "attend": _plain_attend, "logprobs": _plain_logprobs}[op](state)


# ------------------------------------------------------------------------------ 64 bits
def _exact_append(case, s):
    half = DR // 2
    ct, q = s["ct"].double(), s["q"].double()
    lat, rope = s["latent"].double(), s["rope"].double()
    angle = torch.outer(s["positions"].double(), s["inv_freq"].double())
    turn = torch.polar(torch.ones_like(angle), angle)                 # e^(i angle)

    def turned(x, by):
        if case["style"] == "half":
            z = torch.complex(x[..., :half].contiguous(), x[..., half:].contiguous()) * by
            return torch.cat([z.real, z.imag], -1)
        z = torch.view_as_complex(x.reshape(x.shape[:-1] + (half, 2)).contiguous()) * by
        return torch.view_as_real(z).reshape(x.shape)

    new_lat = ct[:, :DL] * torch.rsqrt(ct[:, :DL].pow(2).sum(-1, keepdim=True) / DL + EPS)
    new_lat = new_lat * s["weight"].double()
    new_rope = turned(ct[:, DL:], turn)
    table, page, t = s["table"].tolist(), case["page"], 0
    pages, offsets = [], []
    for b, n in enumerate(s["toks"]):
        for p in range(s["lens_host"][b], s["lens_host"][b] + n):
            pages.append(table[b][p // page])
            offsets.append(p % page)
            t += 1
    pages, offsets = torch.tensor(pages, device=DEV), torch.tensor(offsets, device=DEV)
    lat[pages, offsets] = new_lat
    rope[pages, offsets] = new_rope
    return lat, rope, q[..., :DN].contiguous(), turned(q[..., DN:], turn[:, None])


def _exact_attend(case, s):
    """Keys and values expanded per head, one sequence and eight heads at a time."""
    H, page = case["H"], case["page"]
    out = torch.zeros((s["T"], H, DV), device=DEV, dtype=torch.float64)
    t0 = 0
    for b, n in enumerate(s["toks"]):
        if n == 0:
            continue
        rows = s["lens_host"][b] + n
        used = s["table"][b, : (rows + page - 1) // page].long()
        lat = s["latent"][used].reshape(-1, DL)[:rows].double()
        rope = s["rope"][used].reshape(-1, DR)[:rows].double()
        hidden = torch.zeros((n, rows), device=DEV, dtype=torch.bool)
        for i, w in enumerate(s["mask"][t0: t0 + n].tolist()):
            for j in range(n):
                if not (w >> j) & 1:
                    hidden[i, s["lens_host"][b] + j] = True
        for h in range(0, H, 8):
            k = torch.einsum("rl,hdl->hrd", lat, s["w_uk"][h: h + 8].double())
            v = torch.einsum("rl,hvl->hrv", lat, s["w_uv"][h: h + 8].double())
            a = torch.einsum("thd,hrd->htr", s["q_nope"][t0: t0 + n, h: h + 8].double(), k)
            a += torch.einsum("thd,rd->htr", s["q_rope"][t0: t0 + n, h: h + 8].double(), rope)
            a = (a * s["scale"]).masked_fill_(hidden, float("-inf"))
            out[t0: t0 + n, h: h + 8] = torch.einsum("htr,hrv->thv", torch.softmax(a, -1), v)
        t0 += n
    return out


def _exact_logprobs(case, s):
    G, K = case["G"], case["K"]
    given, entropy, tops = [], [], []
    for r in range(0, case["T"], 128):
        x = s["logits"][r: r + 128].double()
        lp = torch.log_softmax(x, -1)
        p = lp.exp()
        entropy.append(-torch.where(p > 0, p * lp, torch.zeros_like(lp)).sum(-1))
        given.append(lp.gather(1, s["given"][r: r + 128].long()))
        tops.append(lp.topk(K, -1).values)
    T = case["T"]
    return torch.cat(given).view(T, G), torch.cat(entropy), None, torch.cat(tops).view(T, K)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(case, s)
    if case["op"] == "attend":
        return _exact_attend(case, s)
    return _exact_logprobs(case, s)
