"""Caches, pools and 64-bit references for the tests of tree and block-sparse decode (torch on the GPU, plain formulas)."""
import math
import random

import torch

AD, GQA, PAGE, BLOCK = 256, 6, 256, 64
SCALE = 1.0 / 16.0


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


class Store:
    """Rows of B sequences in one contiguous cache (B = 1) or in a page pool, written and read by (sequence, head, position)."""

    def __init__(self, lens, T, nkvh, paged, q8, seed, n_ctx=None, extra_pages=2):
        self.lens, self.T, self.nkvh, self.paged, self.q8, self.B = list(lens), T, nkvh, paged, paged or q8, len(lens)
        self.nqh, r = nkvh * GQA, random.Random(seed)
        assert paged or self.B == 1
        if paged:
            per = [-(-n // PAGE) for n in lens]
            self.max_len = max(max(lens), T)
            self.max_pages = max(1, -(-self.max_len // PAGE))
            self.n_pages = max(1, sum(per) + extra_pages)
            order = list(range(self.n_pages))
            r.shuffle(order)
            table = []
            for n in per:
                table.append([order.pop() for _ in range(n)] + [-1] * (self.max_pages - n))
            self.host_table = table
            self.table, self.seq_len = i32(table), i32(self.lens)
            self.rows = self.n_pages * nkvh * PAGE
        else:
            self.n_ctx = n_ctx or lens[0] + r.randint(0, 70)
            self.pos0 = i32([lens[0] - T])
            self.rows = nkvh * self.n_ctx
            self.max_len = self.n_ctx

    def new(self):
        """A K or V cache (pool) whose every byte is 0xFF: NaN scales, NaN halves."""
        return torch.full((self.rows * (AD + 16 if self.q8 else 2 * AD),), 255, dtype=torch.uint8, device="cuda")

    def index(self, b, h, pos):
        pos = torch.as_tensor(pos, device="cuda").long()
        if not self.paged:
            return h * self.n_ctx + pos
        return (self.table[b].long()[pos // PAGE] * self.nkvh + h) * PAGE + pos % PAGE

    def parts(self, buf):
        if not self.q8:
            return buf.view(torch.float16).view(self.rows, AD), None
        return buf[: self.rows * AD].view(torch.int8).view(self.rows, AD), buf[self.rows * AD:].view(torch.float16).view(self.rows, 8)

    def write(self, buf, b, h, pos, x):
        """x f32 [len(pos)][256]: q8_0 or f16 rows."""
        v, s = self.parts(buf)
        at = self.index(b, h, pos)
        if not self.q8:
            v[at] = x.half()
            return
        x = x.view(-1, 8, 32)
        d = (x.abs().amax(-1, keepdim=True) / 127.0).half().float()
        v[at] = torch.where(d > 0, (x / d).round().clamp(-127, 127), torch.zeros_like(x)).to(torch.int8).view(-1, AD)
        s[at] = d.view(-1, 8).half()

    def write_ints(self, buf, b, h, pos, x):
        """Small whole numbers, stored exactly."""
        v, s = self.parts(buf)
        at = self.index(b, h, pos)
        if self.q8:
            v[at], s[at] = x.to(torch.int8), 1.0
        else:
            v[at] = x.half()

    def read(self, buf, b, h, pos):
        """Stored values in 64 bits."""
        v, s = self.parts(buf)
        at = self.index(b, h, pos)
        x = v[at].double()
        return x if s is None else x * s[at].double().repeat_interleave(32, -1)

    def poison(self, buf, b, h, pos):
        v, s = self.parts(buf)
        at = self.index(b, h, pos)
        if s is None:
            v[at] = float("nan")
        else:
            v[at], s[at] = 127, float("nan")

    def fill(self, buf, g, scale=1.0):
        for b, n in enumerate(self.lens):
            for h in range(self.nkvh):
                if n:
                    self.write(buf, b, h, range(n), torch.randn((n, AD), generator=g, device="cuda") * scale)


def queries(st, seed, scale=1.0):
    g = gen(seed)
    qn = torch.randn((st.B, st.T, st.nqh, AD), generator=g, device="cuda") * scale
    qg = torch.randn((st.B, st.T, st.nqh, 2 * AD), generator=g, device="cuda")
    return qn, qg


def attention(st, kc, vc, qn, qg, visible):
    """visible(b, t, h) -> list of positions. (y, the same with |v|, the largest sum |q k| scale, 1 / sum of P) in 64 bits."""
    y = torch.zeros((st.B, st.T, st.nqh, AD), dtype=torch.float64, device="cuda")
    absy, amax, inv = torch.zeros_like(y), torch.zeros(y.shape[:3], dtype=torch.float64, device="cuda"), torch.zeros(y.shape[:3], dtype=torch.float64, device="cuda")
    for b in range(st.B):
        for t in range(st.T):
            for h in range(st.nkvh):
                pos = visible(b, t, h)
                if len(pos) == 0:
                    continue
                hs = slice(GQA * h, GQA * h + GQA)
                K, V, q = st.read(kc, b, h, pos), st.read(vc, b, h, pos), qn[b, t, hs].double()
                S = q @ K.T * SCALE
                P = torch.exp(S - S.amax(-1, keepdim=True))
                L = P.sum(-1, keepdim=True)
                y[b, t, hs], absy[b, t, hs] = P @ V / L, P @ V.abs() / L
                amax[b, t, hs] = (q.abs() @ K.abs().T * SCALE).amax(-1)
                inv[b, t, hs] = V.abs().amax() * len(pos) / L[:, 0]
    gate = torch.sigmoid(qg[..., AD:].double())
    return y * gate, absy * gate, amax, inv


def check_attention(o, ref, out_eps=2.0 ** -11):
    """|o - y| against the roundings of the kernels, with e(t) = half a step of f16 = 2^-11:
    a score is off by at most 2 e sum|q k| scale (q and k rounded) plus 2^-16 of it (256 f32 additions), so a weight by
    exp(2 * that) - 1; P and V are rounded once each (e each; P below the smallest normal f16 by 2^-25 of the largest P); the
    output is rounded once (out_eps). exp, the sums and the gate in f32: 2^-18 of the sum of the terms' magnitudes.
    The bound assumes the worst sign of every rounding; the norm of the error, in which they are independent, is at most
    2^-9 of the norm of y (score 2^-11.8 for rows of N(0, 1), output 2^-11.8, P and V less)."""
    y, absy, amax, inv = ref
    ds = amax * (2.0 ** -10 + 2.0 ** -16)
    tol = absy * (torch.expm1(2 * ds) + 2.0 ** -10 + 2.0 ** -18)[..., None] if ds.dim() == 3 else None
    tol = tol + (inv * 2.0 ** -25)[..., None] + y.abs() * out_eps + 2.0 ** -25
    d = (o.view(y.shape).double() - y).abs()
    assert torch.isfinite(o.float()).all(), "non-finite values"
    worst = (d - tol).max().item()
    assert worst <= 0, "off by %.3g more than the roundings allow" % worst
    norm = y.norm().item()
    assert d.norm().item() <= 2.0 ** -9 * norm + 1e-6, "relative norm of the error %.3g" % (d.norm().item() / norm)


def tree_visible(st, masks):
    def visible(b, t, h):
        n, m = st.lens[b], masks[b][t]
        base = n - st.T
        return list(range(max(0, base))) + [base + j for j in range(st.T) if (m >> j) & 1 and base + j >= 0]
    return visible


def mask_tensor(masks):
    return torch.tensor([[m - (1 << 64) if m >> 63 else m for m in row] for row in masks], dtype=torch.int64, device="cuda")


def random_masks(B, T, seed, empty=True):
    """Any bits at all (not only trees), bits from T on set too; some rows see no draft."""
    r = random.Random(seed)
    return [[0 if empty and r.random() < 0.1 else r.getrandbits(64) for _ in range(T)] for _ in range(B)]


def call_tree(q27, st, kc, vc, qn, qg, mask, o=None, xq=None, xd=None):
    if o is None and xq is None:
        o = torch.full((st.B, st.T, st.nqh, AD), float("nan"), dtype=torch.float16, device="cuda")
    if st.paged:
        q27.attn_decode_tree_paged(qn, qg, kc, vc, st.table, st.seq_len, mask, o, xq, xd, st.B, st.T, SCALE, st.nqh, st.nkvh,
                                   st.n_pages, st.max_pages, st.max_len)
    else:
        q27.attn_decode_tree(qn, qg, kc, vc, o, xq, xd, st.pos0, mask, st.T, SCALE, st.nqh, st.nkvh, st.n_ctx, st.q8)
    return o


def call_blocks(q27, st, kc, vc, qn, qg, sel, o=None, xq=None, xd=None):
    if o is None and xq is None:
        o = torch.full((st.B, st.T, st.nqh, AD), float("nan"), dtype=torch.float16, device="cuda")
    k = sel.shape[-1]
    if st.paged:
        q27.attn_decode_blocks_paged(qn, qg, kc, vc, st.table, st.seq_len, sel, o, xq, xd, st.B, st.T, k, SCALE, st.nqh, st.nkvh,
                                     st.n_pages, st.max_pages)
    else:
        q27.attn_decode_blocks(qn, qg, kc, vc, o, xq, xd, st.pos0, sel, st.T, k, SCALE, st.nqh, st.nkvh, st.n_ctx, st.q8)
    return o


def call_bounds(q27, st, kc, bounds, T=None):
    T = T or st.T
    if st.paged:
        q27.kv_bounds_paged(kc, bounds, st.table, st.seq_len, st.B, T, st.nkvh, st.n_pages, st.max_pages)
    else:
        q27.kv_bounds(kc, bounds, i32([st.lens[0] - T]), T, st.nkvh, st.n_ctx, st.q8)


def new_bounds(q27, st, fill=float("nan")):
    n = q27.kv_bounds_pool_bytes(st.nkvh, st.n_pages) if st.paged else q27.kv_bounds_bytes(st.nkvh, st.n_ctx)
    return torch.full((n // 2 // (2 * AD), 2, AD), fill, dtype=torch.float16, device="cuda")


def bounds_at(st, b, h, blk):
    """Index of a block's bounds."""
    if st.paged:
        return (st.host_table[b][blk // 4] * st.nkvh + h) * 4 + blk % 4
    return h * (-(-st.n_ctx // BLOCK)) + blk


def call_select(q27, st, qn, bounds, k, sink, recent):
    sel = torch.full((st.B, st.T, st.nkvh, k), -7, dtype=torch.int32, device="cuda")
    if st.paged:
        q27.select_blocks_paged(qn, bounds, sel, st.table, st.seq_len, st.B, st.T, k, sink, recent, st.nqh, st.nkvh, st.n_pages,
                                st.max_pages, st.max_len)
    else:
        q27.select_blocks(qn, bounds, sel, st.pos0, st.T, k, sink, recent, st.nqh, st.nkvh, st.n_ctx)
    return sel


def select_reference(st, qn, bounds, k, sink, recent):
    out = []
    for b, n in enumerate(st.lens):
        for t in range(st.T):
            last = (n - st.T + t) // BLOCK
            for h in range(st.nkvh):
                nb = last + 1
                if nb <= k:
                    out.append(list(range(max(nb, 0))) + [-1] * (k - max(nb, 0)))
                    continue
                at = torch.tensor([bounds_at(st, b, h, i) for i in range(nb)], device="cuda")
                lo, hi = bounds[at, 0].double(), bounds[at, 1].double()
                q = qn[b, t, GQA * h: GQA * h + GQA].double()
                s = (torch.where(q[:, None] < 0, lo, hi) * q[:, None]).sum(-1).amax(0)
                s = torch.where(torch.isnan(s), math.inf, s).tolist()
                must = list(range(sink)) + list(range(nb - recent, nb))
                rest = sorted((i for i in range(sink, nb - recent)), key=lambda i: (-s[i], i))[: k - len(must)]
                out.append(sorted(must + rest))
    return torch.tensor(out, dtype=torch.int32).view(st.B, st.T, st.nkvh, k)
