"""Block-sparse decode: bounds of the keys, choice of blocks, attention over them (q27b_kv_bounds*, q27b_select_blocks*,
q27b_attn_decode_blocks*), and a run of all operators of speculative decoding."""
import random

import pytest
import torch

import helpers_rows as H

pytestmark = pytest.mark.gpu

SHAPES = [
    ([1], 1, 4, False, True), ([4], 4, 1, False, False), ([64], 1, 2, False, True), ([65], 2, 2, False, True),
    ([1003], 4, 4, False, True), ([1003], 3, 2, False, False), ([5000], 1, 4, False, True), ([6401], 4, 1, False, False),
    ([1, 300, 70], 1, 2, True, True), ([700, 4, 1500, 64, 65], 4, 4, True, True), ([5000, 2000], 2, 1, True, True),
]


# ---------------------------------------------------------------- bounds
def reference_bounds(st, kc, bounds, T):
    want = bounds.clone()
    for b, n in enumerate(st.lens):
        for h in range(st.nkvh):
            for blk in range(max(0, n - T) // H.BLOCK, -(-n // H.BLOCK)):
                x = st.read(kc, b, h, range(blk * H.BLOCK, min(n, (blk + 1) * H.BLOCK))).half()
                want[H.bounds_at(st, b, h, blk), 0], want[H.bounds_at(st, b, h, blk), 1] = x.amin(0), x.amax(0)
    return want


@pytest.mark.parametrize("lens,T,nkvh,paged,q8", SHAPES)
@pytest.mark.parametrize("back", ["step", "chunk", "all"])
def test_bounds(q27, lens, T, nkvh, paged, q8, back):
    """The value of a stored row is rounded to f16 once: the smallest and largest are exact. Other blocks stay as they are."""
    st = H.Store(lens, T, nkvh, paged, q8, seed=T)
    kc = st.new()
    st.fill(kc, H.gen(1), 3.0)
    T = {"step": T, "chunk": min(min(lens), 131), "all": min(lens)}[back]
    bounds = H.new_bounds(q27, st, 7.5)
    want = reference_bounds(st, kc, bounds, T)
    H.call_bounds(q27, st, kc, bounds, T)
    assert torch.equal(bounds, want)
    assert q27.device_status() == 0


def test_bounds_of_a_row_that_is_not_finite(q27):
    st = H.Store([200], 1, 1, False, False, seed=1)
    kc = st.new()
    st.fill(kc, H.gen(1))
    v, _ = st.parts(kc)
    v[70, 3], v[71, 4], v[72, 5] = float("nan"), float("inf"), -float("inf")
    bounds = H.new_bounds(q27, st, 0.0)
    H.call_bounds(q27, st, kc, bounds, 200)
    assert torch.isnan(bounds[1, :, 3]).all() and bounds[1, 1, 4] == float("inf") and bounds[1, 0, 5] == -float("inf")
    assert torch.isfinite(bounds[[0, 2, 3]]).all() and torch.isfinite(bounds[1, 0, 4]) and torch.isfinite(bounds[1, 1, 5])


def test_bounds_outside_the_cache(q27):
    st = H.Store([100], 1, 2, False, True, seed=1, n_ctx=130)
    kc = st.new()
    st.fill(kc, H.gen(1))
    for pos, T in ((-50, 40), (130, 5), (-3, 3)):
        bounds = H.new_bounds(q27, st, 7.5)
        q27.kv_bounds(kc, bounds, H.i32([pos]), T, 2, 130)
        assert (bounds == 7.5).all()
    assert q27.device_status() == 0


# ---------------------------------------------------------------- select
@pytest.mark.parametrize("lens,T,nkvh,paged,q8", SHAPES)
@pytest.mark.parametrize("k,sink,recent", [(1, 0, 1), (3, 1, 2), (8, 1, 2), (16, 4, 8), (64, 0, 1), (200, 1, 2)])
def test_select(q27, lens, T, nkvh, paged, q8, k, sink, recent):
    st = H.Store(lens, T, nkvh, paged, q8, seed=T)
    g = H.gen(k)
    bounds = H.new_bounds(q27, st)
    bounds.copy_(torch.randn(bounds.shape, generator=g, device="cuda") + torch.tensor([-2.0, 2.0], device="cuda")[:, None])
    qn, _ = H.queries(st, 3)
    assert torch.equal(H.call_select(q27, st, qn, bounds, k, sink, recent).cpu(), H.select_reference(st, qn, bounds, k, sink, recent))
    assert q27.device_status() == 0


@pytest.mark.parametrize("levels", [1, 2, 5, 40])
@pytest.mark.parametrize("n,k", [(4000, 9), (40000, 31), (70000, 700)])
def test_equal_scores_go_to_the_lower_block(q27, levels, n, k):
    """Whole-number bounds and queries: the scores are exact, and few values are shared by many blocks (0 and -0 among them)."""
    st = H.Store([n], 2, 2, False, True, seed=1)
    r = random.Random(n + levels)
    bounds = H.new_bounds(q27, st, 0.0)
    for i in range(bounds.shape[0]):
        bounds[i, 1, 0] = r.randrange(levels) - levels // 2
        bounds[i, 0, 0] = -40
    qn = torch.zeros((1, 2, st.nqh, H.AD), device="cuda")
    qn[..., 0] = 1.0
    qn[..., 1] = -0.0
    for _ in range(2):
        assert torch.equal(H.call_select(q27, st, qn, bounds, k, 2, 3).cpu(), H.select_reference(st, qn, bounds, k, 2, 3))
        bounds[:, 1, 0].neg_()


def test_scores_next_to_each_other(q27):
    """Blocks whose scores differ in the last bits of a 64-bit sum only are told apart: 1 against 1 + 2^-40."""
    n, nkvh = 64 * 300, 1
    st = H.Store([n], 1, nkvh, False, True, seed=1, n_ctx=n)
    bounds = H.new_bounds(q27, st, 0.0)
    qn = torch.zeros((1, 1, st.nqh, H.AD), device="cuda")
    qn[..., 0], qn[..., 1] = 1.0, 2.0 ** -40
    bounds[:, 1, 0] = 1.0
    better = random.Random(2).sample(range(1, 297), 20)
    bounds[better, 1, 1] = 1.0
    sel = H.call_select(q27, st, qn, bounds, 23, 1, 2)[0, 0, 0].tolist()
    assert sel == [0] + sorted(better) + [298, 299]


def test_a_score_that_is_no_number_wins(q27):
    st = H.Store([64 * 50], 1, 2, False, True, seed=1, n_ctx=64 * 50)
    bounds = H.new_bounds(q27, st, 0.0)
    bounds.copy_(torch.rand(bounds.shape, generator=H.gen(1), device="cuda"))
    bounds[[17, 23], 1, 9] = float("nan")
    bounds[[50 + 30], 1, 9] = float("inf")
    qn = torch.rand((1, 1, st.nqh, H.AD), generator=H.gen(1), device="cuda") + 0.5
    sel = H.call_select(q27, st, qn, bounds, 5, 1, 1)[0, 0].tolist()
    assert {17, 23} < set(sel[0]) and 30 in sel[1]


# ---------------------------------------------------------------- attention over blocks
def block_lists(st, k, seed, holes=True):
    r, out = random.Random(seed), []
    for n in st.lens:
        for t in range(st.T):
            nb = (n - st.T + t) // H.BLOCK + 1
            for _ in range(st.nkvh):
                got = sorted(r.sample(range(nb), r.randint(0 if holes else min(k, nb), min(k, nb)))) if nb > 0 else []
                out.append(got + [-1] * (k - len(got)))
    return torch.tensor(out, dtype=torch.int32).view(st.B, st.T, st.nkvh, k)


def block_visible(st, sel):
    def visible(b, t, h):
        last = st.lens[b] - st.T + t
        return [p for x in sel[b, t, h].tolist() if x >= 0 for p in range(x * H.BLOCK, min((x + 1) * H.BLOCK, last + 1))]
    return visible


@pytest.mark.parametrize("lens,T,nkvh,paged,q8", SHAPES)
@pytest.mark.parametrize("k", [1, 5, 37])
def test_blocks_against_64_bits(q27, lens, T, nkvh, paged, q8, k):
    """Rows of blocks that nobody lists are NaN."""
    st = H.Store(lens, T, nkvh, paged, q8, seed=T)
    kc, vc = st.new(), st.new()
    st.fill(kc, H.gen(1))
    st.fill(vc, H.gen(2))
    sel = block_lists(st, k, seed=k)
    vis = block_visible(st, sel)
    for b, n in enumerate(lens):
        for h in range(nkvh):
            seen = set(p for t in range(T) for p in vis(b, t, h))
            unseen = [p for p in range(n) if p not in seen]
            if unseen:
                st.poison(kc, b, h, unseen)
                st.poison(vc, b, h, unseen)
    qn, qg = H.queries(st, 3)
    o = H.call_blocks(q27, st, kc, vc, qn, qg, sel.cuda())
    H.check_attention(o, H.attention(st, kc, vc, qn, qg, vis))
    assert torch.equal(o, H.call_blocks(q27, st, kc, vc, qn, qg, sel.cuda()))
    assert q27.device_status() == 0


@pytest.mark.parametrize("paged,q8", [(False, True), (False, False), (True, True)])
def test_every_listed_row_counts(q27, paged, q8):
    """q = 0 and whole numbers (see the tree's test): -1 in the middle of a list, a block named twice, lists in any order."""
    st = H.Store([1400] if not paged else [1400, 333], 3, 2, paged, q8, seed=6)
    kc, vc = st.new(), st.new()
    g = H.gen(5)
    for b, n in enumerate(st.lens):
        for h in range(2):
            st.write(kc, b, h, range(n), torch.randn((n, H.AD), generator=g, device="cuda"))
            st.write_ints(vc, b, h, range(n), torch.randint(-4, 5, (n, H.AD), generator=g, device="cuda"))
    r = random.Random(1)
    sel = torch.tensor([[[[r.randrange(-1, -(-n // H.BLOCK)) for _ in range(19)] for _ in range(2)] for _ in range(3)] for n in st.lens],
                       dtype=torch.int32)
    qn = torch.zeros((st.B, 3, st.nqh, H.AD), device="cuda")
    qg = torch.full((st.B, 3, st.nqh, 2 * H.AD), 40.0, device="cuda")
    o = H.call_blocks(q27, st, kc, vc, qn, qg, sel.cuda()).view(st.B, 3, 2, H.GQA, H.AD).double()
    vis = block_visible(st, sel)
    for b in range(st.B):
        for t in range(3):
            for h in range(2):
                pos = vis(b, t, h)
                s = st.read(vc, b, h, pos).sum(0)
                assert s.abs().max() < 1024
                assert torch.equal((o[b, t, h] * len(pos)).round(), s.expand(H.GQA, -1))


@pytest.mark.parametrize("paged,q8", [(False, True), (False, False), (True, True)])
def test_entries_that_are_no_block(q27, paged, q8):
    st = H.Store([500], 2, 2, paged, q8, seed=6)
    kc, vc = st.new(), st.new()
    st.fill(kc, H.gen(1))
    st.fill(vc, H.gen(2))
    qn, qg = H.queries(st, 3)
    good = torch.tensor([0, 3, 7, -1, -1], dtype=torch.int32).expand(1, 2, 2, 5).contiguous()
    want = H.call_blocks(q27, st, kc, vc, qn, qg, good.cuda())
    assert q27.device_status() == 0
    for bad in (-2, -2 ** 31, 2 ** 31 - 1, 2 ** 25, -(-(st.max_pages * 256 if paged else st.n_ctx) // 64)):
        sel = good.clone()
        sel[0, 1, 1, 3] = bad
        assert torch.equal(H.call_blocks(q27, st, kc, vc, qn, qg, sel.cuda()), want)
        assert q27.device_status() == 4
    none = torch.full((1, 2, 2, 5), -1, dtype=torch.int32, device="cuda")
    assert (H.call_blocks(q27, st, kc, vc, qn, qg, none) == 0).all()
    if paged:
        st.table[0, 0] = st.n_pages
        H.call_blocks(q27, st, kc, vc, qn, qg, good.cuda())
        assert q27.device_status() == 2


def test_all_blocks_are_attn_decode(q27):
    st = H.Store([1800], 4, 4, False, True, seed=6)
    kc, vc = st.new(), st.new()
    st.fill(kc, H.gen(1))
    st.fill(vc, H.gen(2))
    qn, qg = H.queries(st, 3)
    sel = torch.arange(-(-1800 // 64), dtype=torch.int32, device="cuda").expand(1, 4, 4, -1).contiguous()
    o = H.call_blocks(q27, st, kc, vc, qn, qg, sel)
    o2 = torch.empty(o.shape, dtype=torch.float32, device="cuda")
    q27.attn_decode(qn, qg, kc, vc, o2, None, None, st.pos0, 4, H.SCALE, 24, 4, st.n_ctx)
    assert ((o.float() - o2).norm() / o2.norm()).item() < 2.0 ** -9


def test_q8_1_output(q27):
    """As the tree's: half a step of d, d rounded to f16, against the f16 output."""
    st = H.Store([500, 77], 2, 2, True, True, seed=8)
    kc, vc = st.new(), st.new()
    st.fill(kc, H.gen(1))
    st.fill(vc, H.gen(2))
    sel = block_lists(st, 4, 1).cuda()
    qn, qg = H.queries(st, 3)
    ob = H.call_blocks(q27, st, kc, vc, qn, qg, sel).double().view(-1, 32)
    xq = torch.zeros(ob.shape, dtype=torch.int8, device="cuda")
    xd = torch.zeros(ob.shape[0], device="cuda")
    H.call_blocks(q27, st, kc, vc, qn, qg, sel, None, xq, xd)
    d = xd.view(-1, 1).double()
    assert ((xq.double() * d - ob).abs() <= d * 0.501 + ob.abs() * 2.0 ** -10 + 1e-7).all()


# ---------------------------------------------------------------- together
@pytest.mark.parametrize("paged", [False, True])
def test_a_speculative_step(q27, paged):
    """Drafting over few blocks, verification of a tree, the accepted path committed, bounds brought up to date; then the next
    draft token. Captured as one graph and replayed."""
    nkvh, T, k = 2, 9, 6
    lens = [1000 + T] if not paged else [1000 + T, 130 + T, 64 + T]
    st = H.Store(lens, T, nkvh, paged, True, seed=6, n_ctx=None if paged else 1100, extra_pages=2)
    kc, vc = st.new(), st.new()
    st.fill(kc, H.gen(1))
    st.fill(vc, H.gen(2))
    g = H.gen(9)
    rn = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    B = st.B
    qg, kr, vr = rn(B, T, st.nqh, 512), rn(B, T, nkvh, 256), rn(B, T, nkvh, 256)
    qw, kw = 1 + 0.1 * rn(256), 1 + 0.1 * rn(256)
    parents = [[-1, 0, 0, 1, 1, 2, 5, 6, 3], [-1, -1, 1, 1, 3, 4, 5, 0, 0], [-1, 0, 1, 2, 3, 4, 5, 6, 7]][:B]
    plans = [q27.tree_plan(p) for p in parents]
    mask = torch.stack([torch.from_numpy(m) for m, _ in plans]).cuda()
    base = torch.tensor([n - T for n in lens], dtype=torch.int32)
    depth = torch.stack([torch.from_numpy(d) for _, d in plans])
    rope3 = (base[:, None] + depth)[..., None].expand(-1, -1, 3).contiguous().cuda()
    path = H.i32([[0, 2, 5, 6, 0, 0, 0, 0, 0], [1, 3, 4, 0, 0, 0, 0, 0, 0], [0, 1, 2, 3, 4, 5, 6, 7, 8]][:B])
    count = H.i32([4, 3, 9][:B])
    qn = torch.zeros((B, T, st.nqh, 256), device="cuda")
    o = torch.zeros((B, T, st.nqh, 256), dtype=torch.float16, device="cuda")
    bounds = H.new_bounds(q27, st, 0.0)
    sel = torch.zeros((B, 1, nkvh, k), dtype=torch.int32, device="cuda")
    q1, g1 = rn(B, 1, st.nqh, 256), rn(B, 1, st.nqh, 512)
    o1 = torch.zeros((B, 1, st.nqh, 256), dtype=torch.float16, device="cuda")
    after = (base + count.cpu()).tolist()  # lengths after the commit; the last row stands for the next token
    pos1, len1 = H.i32([after[0] - 1]), H.i32(after)
    k0, v0 = kc.clone(), vc.clone()

    def step():
        if paged:
            q27.attn_prep_paged(qg, kr, vr, qw, kw, qn, kc, vc, st.table, st.seq_len, B, T, 1e-6, 0.6, st.nqh, nkvh, st.n_pages,
                                st.max_pages, rope3)
        else:
            q27.attn_prep(qg, kr, vr, qw, kw, qn, kc, vc, st.pos0, T, 1e-6, 0.6, st.nqh, nkvh, st.n_ctx, True, rope3)
        H.call_tree(q27, st, kc, vc, qn, qg, mask, o)
        if paged:
            q27.kv_commit_paged(kc, vc, st.table, st.seq_len, path, count, B, T, nkvh, st.n_pages, st.max_pages)
            q27.kv_bounds_paged(kc, bounds, st.table, st.seq_len, B, T, nkvh, st.n_pages, st.max_pages)
            q27.select_blocks_paged(q1, bounds, sel, st.table, len1, B, 1, k, 1, 2, st.nqh, nkvh, st.n_pages, st.max_pages, st.max_len)
            q27.attn_decode_blocks_paged(q1, g1, kc, vc, st.table, len1, sel, o1, None, None, B, 1, k, H.SCALE, st.nqh, nkvh,
                                         st.n_pages, st.max_pages)
        else:
            q27.kv_commit(kc, vc, st.pos0, path, count, T, nkvh, st.n_ctx)
            q27.kv_bounds(kc, bounds, st.pos0, T, nkvh, st.n_ctx)
            q27.select_blocks(q1, bounds, sel, pos1, 1, k, 1, 2, st.nqh, nkvh, st.n_ctx)
            q27.attn_decode_blocks(q1, g1, kc, vc, o1, None, None, pos1, sel, 1, k, H.SCALE, st.nqh, nkvh, st.n_ctx)

    H.call_bounds(q27, st, kc, bounds, min(lens))
    if paged:  # the longer sequences' earlier blocks
        for b in range(B):
            one = q27.kv_bounds_paged
            one(kc, bounds, st.table[b:b + 1], st.seq_len[b:b + 1], 1, lens[b], nkvh, st.n_pages, st.max_pages)
    b0 = bounds.clone()
    step()
    torch.cuda.synchronize()
    masks = [[int(x) & (2 ** 64 - 1) for x in row] for row in mask.tolist()]
    # the tree saw the drafted rows as they were before the commit: write them again to compare
    kd, vd = k0.clone(), v0.clone()
    qn2 = torch.zeros_like(qn)
    if paged:
        q27.attn_prep_paged(qg, kr, vr, qw, kw, qn2, kd, vd, st.table, st.seq_len, B, T, 1e-6, 0.6, st.nqh, nkvh, st.n_pages, st.max_pages, rope3)
    else:
        q27.attn_prep(qg, kr, vr, qw, kw, qn2, kd, vd, st.pos0, T, 1e-6, 0.6, st.nqh, nkvh, st.n_ctx, True, rope3)
    H.check_attention(o, H.attention(st, kd, vd, qn2, qg, H.tree_visible(st, masks)))
    moved = q27.kv_commit_paged if paged else q27.kv_commit
    if paged:
        moved(kd, vd, st.table, st.seq_len, path, count, B, T, nkvh, st.n_pages, st.max_pages)
    else:
        moved(kd, vd, st.pos0, path, count, T, nkvh, st.n_ctx)
    assert torch.equal(kc, kd) and torch.equal(vc, vd)
    st1 = H.Store(after, 1, nkvh, paged, True, seed=6, n_ctx=None if paged else 1100)
    if paged:
        st1.host_table, st1.table, st1.n_pages, st1.rows, st1.max_pages = st.host_table, st.table, st.n_pages, st.rows, st.max_pages
    want = H.select_reference(st1, q1, bounds, k, 1, 2)
    assert torch.equal(sel.cpu(), want)
    H.check_attention(o1, H.attention(st1, kc, vc, q1, g1, block_visible(st1, want)))
    first = [x.clone() for x in (o, kc, vc, bounds, sel, o1)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(2):
        kc.copy_(k0)
        vc.copy_(v0)
        bounds.copy_(b0)
        for x in (o, sel, o1):
            x.zero_()
        graph.replay()
        for x, y in zip((o, kc, vc, bounds, sel, o1), first):
            assert torch.equal(x, y)
    assert q27.device_status() == 0
