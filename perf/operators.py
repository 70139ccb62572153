"""Workloads of the operators around tree verification and block-sparse drafting over a long KV cache.

The model's attention shape: 24 query heads over 4 KV heads of dimension 256 (1 and 2 KV heads: one GPU's share of it).
A cache is q8_0 (int8 values [heads][rows][256], then f16 scales [heads][rows][8]) or f16; a pool has 256-row pages.

  tree    attention of T drafted tokens in the last T rows: every draft sees the prefix and the drafts of its mask
  commit  the rows of the accepted path moved to the front of the drafted rows
  bounds  smallest and largest key per dimension of every 64-row block that the last T rows touch
  select  for every token and KV head the k blocks to attend: the first, the last, and those of the highest bound on q.k
  blocks  attention of T tokens over the rows of such lists of blocks
"""
import importlib
import math
import random

import torch

own = False

AD, GQA, PAGE, BLOCK = 256, 6, 256, 64
KQ_SCALE = 1.0 / 16.0
SINK, RECENT = 1, 2  # blocks at either end that are always attended


def one(kind, name, T, n, nkvh=4, q8=True, k=0):
    """One sequence of n positions in a contiguous cache, the last T of them new."""
    c = {"kind": kind, "paged": False, "T": T, "n": n, "nkvh": nkvh, "q8": q8, "k": k}
    return dict(c, name=name) if name else c


def batch(kind, name, B, T, lo, hi, order, nkvh=4, k=0):
    """B sequences of lo to hi positions, drawn by `order`, over 256-position pages in random order."""
    c = {"kind": kind, "paged": True, "B": B, "T": T, "lo": lo, "hi": hi, "order": order, "nkvh": nkvh, "k": k}
    return dict(c, name=name) if name else c


def listed():
    return [
        # a small tree early in a chat: launches and latency are most of it
        one("tree", "tree_chat", 8, 1003),
        # the widest tree behind a document on an f16 cache, one GPU's quarter of the heads, an odd length
        one("tree", "tree_30k_f16", 64, 30011, nkvh=1, q8=False),
        # an ordinary tree at the longest context
        one("tree", "tree_150k", 16, 150000),
        # verification of a batch of chats of mixed length
        batch("tree", "tree_batch", 16, 12, 64, 16384, 3),
        # the accepted path of one sequence
        one("commit", "commit_chat", 16, 1003),
        # ... and of a full batch of wide trees
        batch("commit", "commit_batch", 64, 64, 128, 4096, 4),
        # the block of a newly appended token
        one("bounds", "bounds_step", 1, 32768),
        # all blocks of a prompt, after its last chunk or when a cache comes back from the host
        one("bounds", "bounds_prompt", 150000, 150000),
        # a draft token at the longest context
        one("select", "select_150k", 1, 150000, k=128),
        # two draft tokens each of a batch of long sequences
        batch("select", "select_batch", 32, 2, 1024, 131072, 5, k=64),
        # attention of that draft token
        one("blocks", "blocks_150k", 1, 150000, k=128),
        # ... and of a batch
        batch("blocks", "blocks_batch", 32, 2, 1024, 32768, 6, k=64),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["tree", "tree", "tree", "commit", "bounds", "select", "blocks", "blocks"])
    nkvh, paged, order = rng.choice([4, 4, 2, 1]), rng.random() < 0.4, rng.randrange(1 << 20)
    q8 = paged or rng.random() < 0.7
    if kind == "tree":
        T = _log(rng, 1, 64)
        if paged:
            B, hi = _log(rng, 1, 16), _log(rng, 256, 8192)
            return batch(kind, None, B, T, max(T, hi // rng.choice([2, 16, 64])), hi, order, nkvh)
        return one(kind, None, T, _log(rng, T, min(150000, 2400000 // T)), nkvh, q8)
    if kind == "commit":
        T = _log(rng, 1, 64)
        if paged:
            return batch(kind, None, _log(rng, 1, 64), T, T, _log(rng, 256, 4096), order, nkvh)
        return one(kind, None, T, _log(rng, T, 32768), nkvh, q8)
    if kind == "bounds":
        if paged:
            T = _log(rng, 1, 2048)
            return batch(kind, None, _log(rng, 1, 32), T, T, _log(rng, 2 * T, 8192), order, nkvh)
        n = _log(rng, 1, 150000)
        return one(kind, None, _log(rng, 1, n), n, nkvh, q8)
    T, k = rng.randint(1, 4), _log(rng, 4, 256)
    if kind == "select":
        if paged:
            hi = _log(rng, 64, 65536)
            return batch(kind, None, _log(rng, 1, 32), T, max(T, hi // rng.choice([2, 32])), hi, order, nkvh, k)
        return one(kind, None, T, _log(rng, T, 150000), nkvh, q8, k)
    if paged:
        hi, k = _log(rng, 64, 16384), min(k, 64)
        return batch(kind, None, _log(rng, 1, 32), T, max(T, hi // rng.choice([2, 32])), hi, order, nkvh, k)
    return one(kind, None, T, _log(rng, T, 150000), nkvh, q8, k)


# ---------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _lengths(case):
    """Lengths of the sequences (they belong to the case, not to the seed)."""
    if not case["paged"]:
        return [case["n"]]
    r = random.Random(case["order"])
    return [r.randint(case["lo"], case["hi"]) for _ in range(case["B"])]


def _rows(rows, gen):
    """Rows of N(0, 1) values around a centre that every 64 rows share: neighbouring tokens are alike."""
    x = torch.randn((rows, AD), generator=gen, device="cuda")
    c = torch.randn((-(-rows // BLOCK), AD), generator=gen, device="cuda")
    return x.add_(c.repeat_interleave(BLOCK, 0)[:rows], alpha=0.5)


def _fill(buf, rows, q8, gen):
    """A cache or pool of `rows` rows in all: q8_0 (d = amax / 127 per 32 values) or f16."""
    step = 1 << 18
    for a in range(0, rows, step):
        b = min(rows, a + step)
        x = _rows(b - a, gen)
        if not q8:
            buf.view(torch.float16).view(rows, AD)[a:b] = x.half()
            continue
        x = x.view(b - a, 8, 32)
        d = x.abs().amax(-1, keepdim=True) / 127.0
        buf[: rows * AD].view(torch.int8).view(rows, AD)[a:b] = (x / d).round_().to(torch.int8).view(b - a, AD)
        buf[rows * AD:].view(torch.float16).view(rows, 8)[a:b] = d.view(b - a, 8).half()


def _cache(rows, q8, gen):
    c = torch.empty(rows * (AD + 16 if q8 else 2 * AD), dtype=torch.uint8, device="cuda")
    _fill(c, rows, q8, gen)
    return c


def _trees(B, T, r):
    """Masks [B][T] of random trees: bit j of token t: draft j is t itself or one of its ancestors."""
    out = []
    for _ in range(B):
        m = []
        for t in range(T):
            p = r.randint(max(-1, t - 6), t - 1)
            m.append((m[p] if p >= 0 else 0) | (1 << t))
        out.append([x - (1 << 64) if x >> 63 else x for x in m])
    return out


def prepare(case, seed):
    gen, r = _gen(seed), random.Random(seed)
    paged, kind, T, nkvh, k = case["paged"], case["kind"], case["T"], case["nkvh"], case["k"]
    nqh, lens = nkvh * GQA, _lengths(case)
    B, q8 = len(lens), paged or case["q8"]
    s = {"case": case, "B": B, "lens": lens, "nqh": nqh, "q8": q8}
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    if paged:
        per = [-(-n // PAGE) for n in lens]
        s["max_pages"], s["n_pages"] = -(-case["hi"] // PAGE), sum(per)
        order = torch.randperm(s["n_pages"], generator=gen, device="cuda").tolist()
        table, at = [], 0
        for n in per:
            table.append(order[at:at + n] + [-1] * (s["max_pages"] - n))
            at += n
        s["table"], s["seq_len"] = i32(table), i32(lens)
        rows = s["n_pages"] * nkvh * PAGE
    else:
        s["n_ctx"] = -(-(case["n"] + 8) // PAGE) * PAGE
        s["pos0"] = i32([case["n"] - T])
        rows = s["n_ctx"] * nkvh
    if kind != "select":
        s["kc"] = _cache(rows, q8, gen)
    if kind in ("tree", "commit", "blocks"):
        s["vc"] = _cache(rows, q8, gen)
    if kind in ("tree", "blocks", "select"):
        lead = (B, T) if paged else (T,)
        s["qn"] = torch.randn((*lead, nqh, AD), generator=gen, device="cuda")
    if kind in ("tree", "blocks"):
        s["qg"] = torch.randn((*lead, nqh, 2 * AD), generator=gen, device="cuda")
        s["o"] = torch.empty((*lead, nqh, AD), dtype=torch.float16, device="cuda")
    if kind == "tree":
        s["mask"] = torch.tensor(_trees(B, T, r), dtype=torch.int64, device="cuda")
    if kind == "commit":
        paths = [sorted(r.sample(range(T), r.randint(1, min(T, 12)))) for _ in range(B)]
        s["count"] = i32([len(p) for p in paths])
        s["path"] = i32([p + [0] * (T - len(p)) for p in paths])
    if kind in ("bounds", "select"):
        s["bounds"] = torch.zeros((rows // BLOCK, 2, AD), dtype=torch.float16, device="cuda")
    if kind == "select":
        step = 1 << 12
        for a in range(0, rows // BLOCK, step):
            b = min(rows // BLOCK, a + step)
            x = _rows((b - a) * BLOCK, gen).view(b - a, BLOCK, AD)
            s["bounds"][a:b, 0], s["bounds"][a:b, 1] = x.amin(1).half(), x.amax(1).half()
        s["sel"] = torch.empty((B, T, nkvh, k), dtype=torch.int32, device="cuda")
    if kind == "blocks":
        sel = []
        for n in lens:
            for t in range(T):
                nb = (n - T + t) // BLOCK + 1
                for _ in range(nkvh):
                    must = set(range(min(SINK, nb))) | set(range(max(0, nb - RECENT), nb))
                    rest = [b for b in r.sample(range(nb), min(nb, k)) if b not in must]
                    got = sorted(sorted(must)[-k:] + rest[: max(0, k - len(must))])
                    sel.append(got + [-1] * (k - len(got)))
        s["sel"] = i32(sel).view(B, T, nkvh, k)
    return s


# ---------------------------------------------------------------- the plain forms
def _views(s, buf):
    """(values, scales or None) of a cache as [pages][heads][rows][..]; a contiguous cache is one page."""
    nkvh = s["case"]["nkvh"]
    o, rows = (s["n_pages"], PAGE) if s["case"]["paged"] else (1, s["n_ctx"])
    if not s["q8"]:
        return buf.view(torch.float16).view(o, nkvh, rows, AD), None
    nv = o * nkvh * rows * AD
    return buf[:nv].view(torch.int8).view(o, nkvh, rows, AD), buf[nv:].view(torch.float16).view(o, nkvh, rows, 8)


def _values(v, d):
    """Stored rows as f32."""
    return v.float() if d is None else (v.float().unflatten(-1, (8, 32)) * d.float().unsqueeze(-1)).flatten(-2)


def _sequences(s, buf, n):
    """The first n rows of every sequence, f32 [B][heads][n][256] (rows past a sequence hold whatever there is)."""
    v, d = _views(s, buf)
    if not s["case"]["paged"]:
        return _values(v[:, :, :n], None if d is None else d[:, :, :n])
    pages = s["table"][:, : -(-n // PAGE)].clamp(min=0).long()
    of = lambda x: x[pages].transpose(1, 2).flatten(2, 3)[:, :, :n]  # noqa: E731
    return _values(of(v), of(d))


def _lens(s):
    return s["seq_len"].long() if s["case"]["paged"] else s["pos0"].long() + s["case"]["T"]


def _gated(s, y):
    """[B][heads][T][6][256] -> the gated output in f16."""
    y = y.permute(0, 2, 1, 3, 4).reshape(s["o"].shape)
    return (y * torch.sigmoid(s["qg"][..., AD:])).half()


def _softmax_v(S, V, eq):
    """Softmax of masked scores times V; 0 where a row has no finite score."""
    P = torch.exp(S - S.amax(-1, keepdim=True).clamp(min=-1e30))
    return torch.einsum(eq, P, V) / P.sum(-1).clamp(min=1e-30).unsqueeze(-1)


def _plain_tree(s):
    T, nkvh, n = s["case"]["T"], s["case"]["nkvh"], max(s["lens"])
    q = s["qn"].view(s["B"], T, nkvh, GQA, AD)
    S = torch.einsum("bthgd,bhnd->bhtgn", q, _sequences(s, s["kc"], n)) * KQ_SCALE
    j = torch.arange(n, device="cuda") - (_lens(s)[:, None] - T)  # [B][n]: number of the draft, < 0 in the prefix
    bit = (s["mask"][:, :, None] >> j.clamp(0, 63)[:, None]) & 1
    seen = (j < 0)[:, None] | ((j < T)[:, None] & (bit == 1))  # [B][T][n]
    S.masked_fill_(~seen[:, None, :, None], -math.inf)
    V = _sequences(s, s["vc"], n)
    V.masked_fill_((j >= T)[:, None, :, None], 0.0)
    return _gated(s, _softmax_v(S, V, "bhtgn,bhnd->bhtgd"))


def _row_index(s, pos):
    """(page, row in it) of positions [B][..]."""
    if not s["case"]["paged"]:
        return torch.zeros_like(pos), pos
    pg = torch.gather(s["table"].long(), 1, (pos // PAGE).flatten(1)).view_as(pos)
    return pg, pos % PAGE


def _plain_commit(s):
    T = s["case"]["T"]
    i = torch.arange(T, device="cuda")[None]
    src = torch.where(i < s["count"][:, None], s["path"].long(), i)
    base = (_lens(s) - T)[:, None]
    (p0, r0), (p1, r1) = _row_index(s, base + src), _row_index(s, base + i)
    k, kd = _views(s, s["kc"])
    v, vd = _views(s, s["vc"])
    k[p1, :, r1] = k[p0, :, r0]
    v[p1, :, r1] = v[p0, :, r0]
    if s["q8"]:
        kd[p1, :, r1] = kd[p0, :, r0]
        vd[p1, :, r1] = vd[p0, :, r0]
    return {"k": s["kc"], "v": s["vc"]}


def _plain_bounds(s):
    T, nkvh, nb = s["case"]["T"], s["case"]["nkvh"], -(-max(s["lens"]) // BLOCK)
    first, end = (_lens(s) - T) // BLOCK * BLOCK, _lens(s)
    # blocks first/64 .. of every sequence, as many as the T rows can touch
    m = min(nb, (T + BLOCK - 2) // BLOCK + 1)
    pos = first[:, None] + torch.arange(m * BLOCK, device="cuda")  # [B][m * 64]
    there = pos < end[:, None]
    pg, row = _row_index(s, torch.where(there, pos, first[:, None]))
    v, d = _views(s, s["kc"])
    x = _values(v[pg, :, row], None if d is None else d[pg, :, row])  # [B][m * 64][heads][256]
    x, there = x.unflatten(1, (m, BLOCK)), there.unflatten(1, (m, BLOCK))
    out = ~there[..., None, None]
    lo, hi = x.masked_fill(out, math.inf).amin(2), x.masked_fill(out, -math.inf).amax(2)  # [B][m][heads][256]
    ok = there[:, :, 0]  # blocks that have a row
    rows_per = PAGE if s["case"]["paged"] else s["n_ctx"]
    at = (pg[:, ::BLOCK, None] * nkvh + torch.arange(nkvh, device="cuda")) * (rows_per // BLOCK) + (row[:, ::BLOCK] // BLOCK)[..., None]
    s["bounds"][at[ok]] = torch.stack([lo[ok], hi[ok]], 2).half()
    return s["bounds"]


def _plain_select(s):
    T, nkvh, k, n = s["case"]["T"], s["case"]["nkvh"], s["case"]["k"], max(s["lens"])
    nb = -(-n // BLOCK)
    if s["case"]["paged"]:
        per = PAGE // BLOCK
        pages = s["table"][:, : -(-nb // per)].clamp(min=0).long()
        bd = s["bounds"].view(s["n_pages"], nkvh, per, 2, AD)[pages].transpose(1, 2).flatten(2, 3)[:, :, :nb]
    else:
        bd = s["bounds"].view(1, nkvh, -1, 2, AD)[:, :, :nb]
    q, bd = s["qn"].view(s["B"], T, nkvh, GQA, AD).double(), bd.double()
    score = torch.einsum("bthgd,bhnd->bthgn", q.clamp(max=0.0), bd[:, :, :, 0])
    score = (score + torch.einsum("bthgd,bhnd->bthgn", q.clamp(min=0.0), bd[:, :, :, 1])).amax(3)
    b = torch.arange(nb, device="cuda")
    last = ((_lens(s)[:, None] - T + torch.arange(T, device="cuda")) // BLOCK)[:, :, None, None]  # a token's own block
    score = torch.where((b < SINK) | (b > last - RECENT), math.inf, score)
    score = torch.where(b > last, -math.inf, score)
    # of equals the first; blocks behind the token's own are no choice, and come last in the list as -1
    got = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :k]
    got = torch.where(got > last, nb, got).sort(-1).values
    got = torch.where(got == nb, -1, got).int()
    return torch.nn.functional.pad(got, (0, k - got.shape[-1]), value=-1)


def _plain_blocks(s):
    T, nkvh, k, B = s["case"]["T"], s["case"]["nkvh"], s["case"]["k"], s["B"]
    sel = s["sel"].long()  # [B][T][heads][k]
    pos = (sel.clamp(min=0)[..., None] * BLOCK + torch.arange(BLOCK, device="cuda")).flatten(3)
    q_pos = (_lens(s)[:, None] - T + torch.arange(T, device="cuda"))[:, :, None, None]
    seen = (pos <= q_pos) & (sel >= 0).repeat_interleave(BLOCK, -1)
    pg, row = _row_index(s, torch.where(seen, pos, 0))
    h = torch.arange(nkvh, device="cuda")[:, None]
    (kv, kd), (vv, vd) = _views(s, s["kc"]), _views(s, s["vc"])
    K = _values(kv[pg, h, row], None if kd is None else kd[pg, h, row])
    S = torch.einsum("bthgd,bthnd->bhtgn", s["qn"].view(B, T, nkvh, GQA, AD), K) * KQ_SCALE
    S.masked_fill_(~seen.transpose(1, 2)[:, :, :, None], -math.inf)
    del K
    V = _values(vv[pg, h, row], None if vd is None else vd[pg, h, row])
    return _gated(s, _softmax_v(S, V, "bhtgn,bthnd->bhtgd"))


# ---------------------------------------------------------------- the framework's calls
def _call(s):
    q27 = importlib.import_module("qwen27-engine_b200")
    c, T, nkvh, nqh, k, B = s["case"], s["case"]["T"], s["case"]["nkvh"], s["nqh"], s["case"]["k"], s["B"]
    if c["paged"]:
        hi, np_, mp = c["hi"], s["n_pages"], s["max_pages"]
        if c["kind"] == "tree":
            q27.attn_decode_tree_paged(s["qn"], s["qg"], s["kc"], s["vc"], s["table"], s["seq_len"], s["mask"], s["o"], None, None,
                                       B, T, KQ_SCALE, nqh, nkvh, np_, mp, hi)
        elif c["kind"] == "commit":
            q27.kv_commit_paged(s["kc"], s["vc"], s["table"], s["seq_len"], s["path"], s["count"], B, T, nkvh, np_, mp)
        elif c["kind"] == "bounds":
            q27.kv_bounds_paged(s["kc"], s["bounds"], s["table"], s["seq_len"], B, T, nkvh, np_, mp)
        elif c["kind"] == "select":
            q27.select_blocks_paged(s["qn"], s["bounds"], s["sel"], s["table"], s["seq_len"], B, T, k, SINK, RECENT, nqh, nkvh, np_, mp,
                                    hi)
        else:
            q27.attn_decode_blocks_paged(s["qn"], s["qg"], s["kc"], s["vc"], s["table"], s["seq_len"], s["sel"], s["o"], None, None,
                                         B, T, k, KQ_SCALE, nqh, nkvh, np_, mp)
    elif c["kind"] == "tree":
        q27.attn_decode_tree(s["qn"], s["qg"], s["kc"], s["vc"], s["o"], None, None, s["pos0"], s["mask"], T, KQ_SCALE, nqh, nkvh,
                             s["n_ctx"], s["q8"])
    elif c["kind"] == "commit":
        q27.kv_commit(s["kc"], s["vc"], s["pos0"], s["path"], s["count"], T, nkvh, s["n_ctx"], s["q8"])
    elif c["kind"] == "bounds":
        q27.kv_bounds(s["kc"], s["bounds"], s["pos0"], T, nkvh, s["n_ctx"], s["q8"])
    elif c["kind"] == "select":
        q27.select_blocks(s["qn"], s["bounds"], s["sel"], s["pos0"], T, k, SINK, RECENT, nqh, nkvh, s["n_ctx"])
    else:
        q27.attn_decode_blocks(s["qn"], s["qg"], s["kc"], s["vc"], s["o"], None, None, s["pos0"], s["sel"], T, k, KQ_SCALE, nqh, nkvh,
                               s["n_ctx"], s["q8"])
    if c["kind"] == "commit":
        return {"k": s["kc"], "v": s["vc"]}
    return {"tree": s.get("o"), "bounds": s.get("bounds"), "select": s.get("sel"), "blocks": s.get("o")}[c["kind"]]


def run(state):
    if own:
        return _call(state)
    return {"tree": _plain_tree, "commit": _plain_commit, "bounds": _plain_bounds, "select": _plain_select,
            "blocks": _plain_blocks}[state["case"]["kind"]](state)


# ---------------------------------------------------------------- the definition in 64 bits
def _exact_rows(s, buf, b, h, pos):
    """Rows `pos` of head h of sequence b in 64 bits."""
    nkvh = s["case"]["nkvh"]
    if s["case"]["paged"]:
        idx = (s["table"][b].long()[pos // PAGE] * nkvh + h) * PAGE + pos % PAGE
        rows = s["n_pages"] * nkvh * PAGE
    else:
        idx = h * s["n_ctx"] + pos
        rows = s["n_ctx"] * nkvh
    if not s["q8"]:
        return buf.view(torch.float16).view(rows, AD)[idx].double()
    x = buf[: rows * AD].view(torch.int8).view(rows, AD)[idx].double()
    return x * buf[rows * AD:].view(torch.float16).view(rows, 8)[idx].double().repeat_interleave(32, -1)


def exact(case, seed):
    if case["kind"] in ("commit", "select"):
        return None  # moved bytes, and whole numbers
    s = prepare(case, seed)
    T, nkvh = case["T"], case["nkvh"]
    if case["kind"] == "bounds":
        out = s["bounds"].double()
        for b, n in enumerate(s["lens"]):
            for h in range(nkvh):
                lo = (n - T) // BLOCK
                pos = torch.arange(lo * BLOCK, n, device="cuda")
                x = _exact_rows(s, s["kc"], b, h, pos)
                blk = torch.arange(lo, -(-n // BLOCK), device="cuda")
                if case["paged"]:
                    at = (s["table"][b].long()[blk // 4] * nkvh + h) * 4 + blk % 4
                else:
                    at = h * (s["n_ctx"] // BLOCK) + blk
                full = len(x) // BLOCK
                whole = x[: full * BLOCK].view(full, BLOCK, AD)
                out[at[:full], 0], out[at[:full], 1] = whole.amin(1), whole.amax(1)
                if full < len(blk):
                    out[at[full], 0], out[at[full], 1] = x[full * BLOCK:].amin(0), x[full * BLOCK:].amax(0)
        return out
    out = torch.zeros((s["B"], T, s["nqh"], AD), dtype=torch.float64, device="cuda")
    masks = s["mask"].tolist() if case["kind"] == "tree" else None
    qn, qg = s["qn"].view(out.shape).double(), s["qg"].view(s["B"], T, s["nqh"], 2 * AD).double()
    for b, n in enumerate(s["lens"]):
        for h in range(nkvh):
            heads = slice(GQA * h, GQA * h + GQA)
            if case["kind"] == "tree":
                pos = torch.arange(n, device="cuda")
                K, V = _exact_rows(s, s["kc"], b, h, pos), _exact_rows(s, s["vc"], b, h, pos)
            for t in range(T):
                if case["kind"] == "tree":
                    drafts = [j for j in range(T) if (masks[b][t] >> j) & 1]
                    at = torch.cat([pos[: n - T], n - T + torch.tensor(drafts, dtype=torch.long, device="cuda")])
                    w = torch.zeros(n, dtype=torch.bool, device="cuda")
                    w[at] = True
                    score = (qn[b, t, heads] @ K.T * KQ_SCALE).masked_fill(~w, -math.inf)
                    out[b, t, heads] = torch.softmax(score, -1) @ V
                    continue
                blk = s["sel"][b, t, h].long()
                at = (blk[blk >= 0][:, None] * BLOCK + torch.arange(BLOCK, device="cuda")).flatten()
                at = at[at <= n - T + t]
                K, V = _exact_rows(s, s["kc"], b, h, at), _exact_rows(s, s["vc"], b, h, at)
                out[b, t, heads] = torch.softmax(qn[b, t, heads] @ K.T * KQ_SCALE, -1) @ V
    return (out * torch.sigmoid(qg[..., AD:])).view(s["o"].shape)


# ---------------------------------------------------------------- bytes and operations that a pass cannot do without
def work(case):
    lens, T, nkvh, k = _lengths(case), case["T"], case["nkvh"], case["k"]
    row = AD + 16 if case["paged"] or case["q8"] else 2 * AD
    B, N, nqh = len(lens), sum(lens), nkvh * GQA
    io = B * T * nqh * AD * (4 + 4 + 2)  # query, gate, output
    if case["kind"] == "tree":
        return {"bytes": 2 * N * nkvh * row + io + 8 * B * T, "flops": 4 * T * nqh * AD * N}
    if case["kind"] == "commit":
        return {"bytes": 2 * 2 * B * min(T, 12) // 2 * nkvh * row, "flops": 0}
    if case["kind"] == "bounds":
        blocks = [-(-n // BLOCK) - (n - T) // BLOCK for n in lens]
        rows = sum(n - (n - T) // BLOCK * BLOCK for n in lens)
        return {"bytes": nkvh * (rows * row + sum(blocks) * 4 * AD), "flops": 2 * rows * nkvh * AD}
    nb = [-(-n // BLOCK) for n in lens]
    if case["kind"] == "select":
        return {"bytes": sum(nb) * nkvh * 4 * AD + B * T * (nqh * AD * 4 + nkvh * k * 4), "flops": 2 * T * nqh * AD * sum(nb)}
    rows = sum(min(n, min(k, x) * BLOCK) for n, x in zip(lens, nb)) * T
    return {"bytes": 2 * rows * nkvh * row + io + 4 * B * T * nkvh * k, "flops": 4 * rows * nqh * AD}
