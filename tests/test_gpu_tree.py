"""Attention of a tree of drafts, and the accepted path moved to the front (q27b_attn_decode_tree*, q27b_kv_commit*)."""
import random

import pytest
import torch

import helpers_rows as H

pytestmark = pytest.mark.gpu

# (lengths with the drafts, T, KV heads, paged, q8)
SHAPES = [
    ([1], 1, 4, False, True), ([8], 8, 1, False, True), ([64], 64, 2, False, True), ([65], 1, 1, False, False),
    ([300], 5, 4, False, True), ([1003], 8, 4, False, True), ([1003], 21, 4, False, False), ([700], 22, 3, False, True),
    ([2000], 64, 4, False, True), ([1999], 43, 1, False, False), ([4160], 16, 4, False, True), ([129], 64, 4, False, False),
    ([5, 300, 70, 1], 1, 2, True, True), ([12, 257, 1000, 64, 640], 12, 4, True, True), ([64, 900], 64, 1, True, True),
    ([2100, 33, 1500], 22, 4, True, True),
]


def counted(st, vals, visible):
    """Sums of whole-number V rows over the visible rows, and how many there are."""
    s = torch.zeros((st.B, st.T, st.nkvh, H.AD), dtype=torch.float64, device="cuda")
    n = torch.zeros((st.B, st.T, st.nkvh, 1), dtype=torch.float64, device="cuda")
    for b in range(st.B):
        for t in range(st.T):
            for h in range(st.nkvh):
                pos = visible(b, t, h)
                n[b, t, h] = len(pos)
                if pos:
                    s[b, t, h] = st.read(vals, b, h, pos).sum(0)
    return s, n


@pytest.mark.parametrize("lens,T,nkvh,paged,q8", SHAPES)
def test_every_visible_row_counts_once(q27, lens, T, nkvh, paged, q8):
    """q = 0: every weight is 1 / n exactly, and y n is the sum of whole numbers |v| <= 4: rounded to f16 it is off by less
    than a half while |sum| < 1024 (here below 4 sqrt(n) * 6), so every missing or extra row shows. What no draft sees is NaN."""
    st = H.Store(lens, T, nkvh, paged, q8, seed=len(lens) * 100 + T)
    kc, vc = st.new(), st.new()
    masks = H.random_masks(st.B, T, seed=T)
    g = H.gen(5)
    for b, n in enumerate(lens):
        for h in range(nkvh):
            st.write(kc, b, h, range(n), torch.randn((n, H.AD), generator=g, device="cuda"))
            st.write_ints(vc, b, h, range(n), torch.randint(-4, 5, (n, H.AD), generator=g, device="cuda"))
            seen = 0
            for m in masks[b]:
                seen |= m
            for j in range(T):
                if not (seen >> j) & 1:
                    st.poison(kc, b, h, [n - T + j])
                    st.poison(vc, b, h, [n - T + j])
    qn = torch.zeros((st.B, T, st.nqh, H.AD), device="cuda")
    qg = torch.full((st.B, T, st.nqh, 2 * H.AD), 40.0, device="cuda")
    o = H.call_tree(q27, st, kc, vc, qn, qg, H.mask_tensor(masks))
    s, n = counted(st, vc, H.tree_visible(st, masks))
    got = o.double().view(st.B, T, nkvh, H.GQA, H.AD) * n[..., None, :]
    assert s.abs().max() < 1024
    assert torch.equal(got.round(), s[:, :, :, None].expand_as(got))
    assert torch.equal(o.view(st.B, T, nkvh, H.GQA, H.AD)[(n[..., 0] == 0)], torch.zeros_like(o.view(st.B, T, nkvh, H.GQA, H.AD)[(n[..., 0] == 0)]))
    assert q27.device_status() == 0


@pytest.mark.parametrize("lens,T,nkvh,paged,q8", SHAPES)
def test_against_64_bits(q27, lens, T, nkvh, paged, q8):
    st = H.Store(lens, T, nkvh, paged, q8, seed=len(lens) * 10 + T)
    kc, vc = st.new(), st.new()
    st.fill(kc, H.gen(1))
    st.fill(vc, H.gen(2))
    masks = H.random_masks(st.B, T, seed=T + 1)
    qn, qg = H.queries(st, 3)
    ref = H.attention(st, kc, vc, qn, qg, H.tree_visible(st, masks))
    o = H.call_tree(q27, st, kc, vc, qn, qg, H.mask_tensor(masks))
    H.check_attention(o, ref)
    again = H.call_tree(q27, st, kc, vc, qn, qg, H.mask_tensor(masks))
    assert torch.equal(o, again)  # the same bits on every run


@pytest.mark.parametrize("big", [1, 40])
def test_scores_that_run_away(q27, big):
    """Rows whose maximum keeps moving: scores that grow along the sequence, up to a one-hot softmax."""
    st = H.Store([900], 9, 2, False, True, seed=1)
    kc, vc = st.new(), st.new()
    for h in range(2):
        base = torch.randn((1, H.AD), generator=H.gen(h), device="cuda")
        ramp = torch.linspace(-1, 1, 900, device="cuda")[:, None] * big
        st.write(kc, 0, h, range(900), base * ramp)
    st.fill(vc, H.gen(2))
    masks = H.random_masks(1, 9, seed=4, empty=False)
    qn, qg = H.queries(st, 3)
    ref = H.attention(st, kc, vc, qn, qg, H.tree_visible(st, masks))
    o = H.call_tree(q27, st, kc, vc, qn, qg, H.mask_tensor(masks)).view(ref[0].shape).double()
    ds = ref[2] * (2.0 ** -10 + 2.0 ** -16)
    tol = ref[1] * (torch.expm1(2 * ds) + 2.0 ** -10)[..., None] + (ref[3] * 2.0 ** -25)[..., None] + ref[0].abs() * 2.0 ** -11 + 2.0 ** -25
    assert ((o - ref[0]).abs() <= tol).all()


@pytest.mark.parametrize("paged,q8", [(False, True), (False, False), (True, True)])
def test_infinities_and_nan_stay_with_the_drafts_that_see_them(q27, paged, q8):
    """Draft rows that hold NaN or overflow: a draft that does not see them is exact, one that does is not finite."""
    T, n = 11, 390
    st = H.Store([n], T, 2, paged, q8, seed=3)
    kc, vc = st.new(), st.new()
    st.fill(kc, H.gen(1))
    st.fill(vc, H.gen(2))
    masks = [[(1 << t) | (1 << 0) if t % 2 else 1 << t for t in range(T)]]  # odd drafts see draft 0 and themselves
    qn, qg = H.queries(st, 3)
    clean = H.call_tree(q27, st, kc, vc, qn, qg, H.mask_tensor(masks))
    for which in ("k", "v"):
        k2, v2 = kc.clone(), vc.clone()
        for h in range(2):
            st.poison(k2 if which == "k" else v2, 0, h, [n - T])
        o = H.call_tree(q27, st, k2, v2, qn, qg, H.mask_tensor(masks))[0]
        for t in range(T):
            if t == 0 or t % 2:
                assert torch.isnan(o[t]).all(), (which, t)
            else:
                assert torch.equal(o[t], clean[0][t]), (which, t)


def test_a_chain_is_attn_decode(q27):
    st = H.Store([700], 4, 4, False, True, seed=8)
    kc, vc = st.new(), st.new()
    st.fill(kc, H.gen(1))
    st.fill(vc, H.gen(2))
    mask, depth = q27.tree_plan([-1, 0, 1, 2])
    assert depth.tolist() == [0, 1, 2, 3]
    qn, qg = H.queries(st, 3)
    o = H.call_tree(q27, st, kc, vc, qn, qg, torch.from_numpy(mask).cuda().view(1, -1))
    o2 = torch.empty(o.shape, dtype=torch.float32, device="cuda")
    q27.attn_decode(qn, qg, kc, vc, o2, None, None, st.pos0, 4, H.SCALE, 24, 4, st.n_ctx)
    assert ((o.float() - o2).norm() / o2.norm()).item() < 2.0 ** -9


@pytest.mark.parametrize("paged", [False, True])
def test_q8_1_output(q27, paged):
    """xq xd is the same result: d = amax / 127 and half a step of it, and d itself rounded to f16 (2^-11 of |y|), against the
    f16 output (2^-11 of |y|)."""
    st = H.Store([500] if not paged else [500, 77], 7, 2, paged, True, seed=8)
    kc, vc = st.new(), st.new()
    st.fill(kc, H.gen(1))
    st.fill(vc, H.gen(2))
    mask = H.mask_tensor(H.random_masks(st.B, 7, seed=9))
    qn, qg = H.queries(st, 3)
    o = H.call_tree(q27, st, kc, vc, qn, qg, mask).double()
    xq = torch.zeros(o.shape, dtype=torch.int8, device="cuda")
    xd = torch.zeros(o.numel() // 32, device="cuda")
    H.call_tree(q27, st, kc, vc, qn, qg, mask, None, xq, xd)
    d = xd.view(-1, 1).double()
    y = xq.view(-1, 32).double() * d
    ob = o.view(-1, 32)
    assert ((y - ob).abs() <= d * 0.501 + ob.abs() * 2.0 ** -10 + 1e-7).all()
    amax = ob.abs().amax(-1, keepdim=True)
    assert ((d * 127 - amax).abs() <= amax * 2.0 ** -10 + 1e-5).all()


def test_sequences_of_no_length(q27):
    """seq_len 0 and below T in a batch: what is there is attended, the rest gives 0."""
    st = H.Store([0, 3, 300], 5, 2, True, True, seed=2)
    kc, vc = st.new(), st.new()
    st.fill(kc, H.gen(1))
    st.fill(vc, H.gen(2))
    masks = [[0b11111] * 5] * 3
    qn, qg = H.queries(st, 3)
    o = H.call_tree(q27, st, kc, vc, qn, qg, H.mask_tensor(masks))
    assert (o[0] == 0).all()
    H.check_attention(o, H.attention(st, kc, vc, qn, qg, H.tree_visible(st, masks)))


def test_bad_pages_are_reported(q27):
    st = H.Store([700, 300], 6, 2, True, True, seed=2)
    kc, vc = st.new(), st.new()
    st.fill(kc, H.gen(1))
    st.fill(vc, H.gen(2))
    mask = H.mask_tensor(H.random_masks(2, 6, seed=9))
    qn, qg = H.queries(st, 3)
    want = H.call_tree(q27, st, kc, vc, qn, qg, mask)
    for bad in (-5, st.n_pages, 2 ** 31 - 1):
        st.table[0, 1] = bad
        o = H.call_tree(q27, st, kc, vc, qn, qg, mask)
        assert q27.device_status() == 2
        assert torch.equal(o[1], want[1])
    assert q27.device_status() == 0


def test_replayed_graph_sees_new_positions_and_masks(q27):
    T, nkvh = 13, 4
    st = H.Store([1500], T, nkvh, False, True, seed=4)
    kc, vc = st.new(), st.new()
    st.fill(kc, H.gen(1))
    st.fill(vc, H.gen(2))
    qn, qg = H.queries(st, 3)
    mask = H.mask_tensor(H.random_masks(1, T, seed=1))
    o = torch.zeros((1, T, st.nqh, H.AD), dtype=torch.float16, device="cuda")
    H.call_tree(q27, st, kc, vc, qn, qg, mask, o)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        H.call_tree(q27, st, kc, vc, qn, qg, mask, o)
    for n, seed in ((1500, 1), (T, 2), (64, 3), (777, 4)):
        masks = H.random_masks(1, T, seed=seed)
        st.lens = [n]
        st.pos0.fill_(n - T)
        mask.copy_(H.mask_tensor(masks))
        graph.replay()
        H.check_attention(o, H.attention(st, kc, vc, qn, qg, H.tree_visible(st, masks)))


def test_on_another_stream(q27):
    st = H.Store([900], 17, 2, False, True, seed=4)
    kc, vc = st.new(), st.new()
    st.fill(kc, H.gen(1))
    st.fill(vc, H.gen(2))
    mask = H.mask_tensor(H.random_masks(1, 17, seed=1))
    qn, qg = H.queries(st, 3)
    want = H.call_tree(q27, st, kc, vc, qn, qg, mask)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        qn2 = torch.zeros_like(qn)
        for _ in range(20):  # still being written when the call is made
            qn2.add_(qn, alpha=0.05)
        qn2.copy_(qn)
        o = H.call_tree(q27, st, kc, vc, qn2, qg, mask)
    side.synchronize()
    assert torch.equal(o, want)


# ---------------------------------------------------------------- commit
def committed(st, buf, paths, counts):
    want = buf.clone()
    v, s = st.parts(buf)
    wv, ws = st.parts(want)
    for b, n in enumerate(st.lens):
        for i in range(max(0, min(counts[b], st.T))):
            f = paths[b][i]
            if f < 0 or f >= st.T:
                continue
            for h in range(st.nkvh):
                src, dst = st.index(b, h, [n - st.T + f]), st.index(b, h, [n - st.T + i])
                wv[dst] = v[src]
                if s is not None:
                    ws[dst] = s[src]
    return want


@pytest.mark.parametrize("lens,T,nkvh,paged,q8", SHAPES)
@pytest.mark.parametrize("how", ["path", "any"])
def test_commit(q27, lens, T, nkvh, paged, q8, how):
    st = H.Store(lens, T, nkvh, paged, q8, seed=T)
    if min(lens) < T:
        pytest.skip("drafts before the sequence")
    r = random.Random(T)
    kc, vc = st.new(), st.new()
    st.fill(kc, H.gen(1))
    st.fill(vc, H.gen(2))
    counts = [r.choice([0, 1, T, r.randint(0, T), T + 3 if how == "any" else T]) for _ in lens]
    if how == "path":
        paths = [sorted(r.sample(range(T), min(T, max(c, 0)))) + [0] * (T - min(T, max(c, 0))) for c in counts]
    else:  # any order, the same row twice
        paths = [[r.randrange(T) for _ in range(T)] for _ in counts]
    want = committed(st, kc, paths, counts), committed(st, vc, paths, counts)
    if paged:
        q27.kv_commit_paged(kc, vc, st.table, st.seq_len, H.i32(paths), H.i32(counts), st.B, T, nkvh, st.n_pages, st.max_pages)
    else:
        q27.kv_commit(kc, vc, st.pos0, H.i32(paths[0]), H.i32(counts), T, nkvh, st.n_ctx, q8)
    assert torch.equal(kc, want[0]) and torch.equal(vc, want[1])
    assert q27.device_status() == 0


def test_commit_reports_what_is_no_draft(q27):
    st = H.Store([100], 6, 2, False, True, seed=1)
    kc, vc = st.new(), st.new()
    st.fill(kc, H.gen(1))
    st.fill(vc, H.gen(2))
    paths = [[3, -1, 6, 5, 2 ** 30, 0]]
    want = committed(st, kc, paths, [5]), committed(st, vc, paths, [5])
    q27.kv_commit(kc, vc, st.pos0, H.i32(paths[0]), H.i32([5]), 6, 2, st.n_ctx)
    assert q27.device_status() == 4
    assert torch.equal(kc, want[0]) and torch.equal(vc, want[1])
    # rows outside the cache are left alone
    before = kc.clone()
    for pos in (-4, st.n_ctx - 2):
        q27.kv_commit(kc, vc, H.i32([pos]), H.i32([5, 4, 3, 2, 1, 0]), H.i32([3]), 6, 2, st.n_ctx)
        v, s = st.parts(kc)
        bv, bs = st.parts(before)
        ok = [r for r in range(st.rows) if not any(0 <= pos + i < st.n_ctx and 0 <= pos + 5 - i < st.n_ctx and r % st.n_ctx == pos + i for i in range(3))]
        assert torch.equal(v[ok], bv[ok])
        kc.copy_(before)
    assert q27.device_status() == 0


# ---------------------------------------------------------------- memory
def test_rows_far_behind_2_to_the_31_bytes(q27):
    """Pages at both ends of a pool of 2.7 GB: addresses and row numbers that 32 bits of bytes do not reach."""
    n_pages, nkvh, T = 39000, 1, 7
    st = H.Store([600], T, nkvh, True, True, seed=1, extra_pages=0)
    st.n_pages, st.rows = n_pages, n_pages * nkvh * H.PAGE
    st.host_table = [[n_pages - 1, 0, n_pages - 17]]
    st.table = H.i32(st.host_table)
    kc, vc = (torch.empty(st.rows * (H.AD + 16), dtype=torch.uint8, device="cuda") for _ in range(2))
    assert kc.numel() > 2 ** 31
    st.fill(kc, H.gen(1))
    st.fill(vc, H.gen(2))
    masks = H.random_masks(1, T, seed=2)
    qn, qg = H.queries(st, 3)
    o = H.call_tree(q27, st, kc, vc, qn, qg, H.mask_tensor(masks))
    H.check_attention(o, H.attention(st, kc, vc, qn, qg, H.tree_visible(st, masks)))
    rows = lambda buf, pos: tuple(x.clone() for x in (st.parts(buf)[0][st.index(0, 0, pos)], st.parts(buf)[1][st.index(0, 0, pos)]))  # noqa: E731
    want = [rows(c, [600 - T + 3, 600 - T + 5]) for c in (kc, vc)]
    q27.kv_commit_paged(kc, vc, st.table, st.seq_len, H.i32([[3, 5, 0, 0, 0, 0, 0]]), H.i32([2]), 1, T, nkvh, n_pages, st.max_pages)
    got = [rows(c, [600 - T, 600 - T + 1]) for c in (kc, vc)]
    for a, b in zip(want, got):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    bounds = torch.full((n_pages * 4, 2, H.AD), 7.5, dtype=torch.float16, device="cuda")
    H.call_bounds(q27, st, kc, bounds, 600)
    for blk in range(10):
        x = st.read(kc, 0, 0, range(64 * blk, min(600, 64 * blk + 64))).half()
        i = H.bounds_at(st, 0, 0, blk)
        assert torch.equal(bounds[i, 0], x.amin(0)) and torch.equal(bounds[i, 1], x.amax(0))
    st1 = H.Store([600], 1, nkvh, True, True, seed=1, extra_pages=0)
    st1.n_pages, st1.rows, st1.table, st1.host_table = n_pages, st.rows, st.table, st.host_table
    q1, g1 = H.queries(st1, 4)
    sel = H.call_select(q27, st1, q1, bounds, 5, 1, 2)
    assert torch.equal(sel.cpu(), H.select_reference(st1, q1, bounds, 5, 1, 2))
    o = H.call_blocks(q27, st1, kc, vc, q1, g1, sel)
    pos = lambda b, t, h: [p for x in sel[0, 0, h].tolist() for p in range(64 * x, min(64 * x + 64, 600))]  # noqa: E731
    H.check_attention(o, H.attention(st1, kc, vc, q1, g1, pos))
    assert q27.device_status() == 0


def test_small_and_fixed_workspaces(q27):
    """A prefill buffer that holds fewer parts gives the same result; one that holds none, and a paged buffer that is fixed and
    too small, are refused with the caller's name. A paged buffer that grows leaves what a captured graph names in place."""
    T = 9
    st = H.Store([1500], T, 2, False, True, seed=4)
    pg = H.Store([1500, 700], T, 2, True, True, seed=4)
    sets = []
    for s in (st, pg):
        kc, vc = s.new(), s.new()
        s.fill(kc, H.gen(1))
        s.fill(vc, H.gen(2))
        masks = H.random_masks(s.B, T, seed=1)
        qn, qg = H.queries(s, 3)
        sets.append((s, kc, vc, qn, qg, H.mask_tensor(masks), H.attention(s, kc, vc, qn, qg, H.tree_visible(s, masks))))
    sel = torch.tensor([[[[0, 3, 9], [1, 2, 3]]]], dtype=torch.int32, device="cuda")
    st1 = H.Store([1500], 1, 2, False, True, seed=4, n_ctx=st.n_ctx)
    try:
        q27.workspace_destroy()
        q27.workspace_init(2 * 3 * 128 * 258 * 4 + 64, 4096)  # three parts for each of the two units
        H.check_attention(H.call_tree(q27, *sets[0][:6]), sets[0][6])
        with pytest.raises(q27.Q27Error, match="attn_decode_tree_paged.*fixed"):
            H.call_tree(q27, *sets[1][:6])
        q27.workspace_destroy()
        q27.workspace_init(4096, 0)
        with pytest.raises(q27.Q27Error, match="attn_decode_tree: the prefill workspace is too small"):
            H.call_tree(q27, *sets[0][:6])
        with pytest.raises(q27.Q27Error, match="attn_decode_blocks: the prefill workspace is too small"):
            H.call_blocks(q27, st1, sets[0][1], sets[0][2], sets[0][3][:, :1].contiguous(), sets[0][4][:, :1].contiguous(), sel)
        q27.workspace_destroy()
        # over pages: a graph, then a call that needs more
        o = H.call_tree(q27, *sets[1][:6])
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            H.call_tree(q27, *sets[1][:6], o)
        before = q27.workspace_query()[2]
        big = H.Store([300] * 40, 64, 4, True, True, seed=4)
        kb, vb = big.new(), big.new()
        big.fill(kb, H.gen(1))
        big.fill(vb, H.gen(2))
        qn, qg = H.queries(big, 3)
        H.call_tree(q27, big, kb, vb, qn, qg, H.mask_tensor(H.random_masks(40, 64, seed=1)))
        assert q27.workspace_query()[2] > before
        o.zero_()
        graph.replay()
        H.check_attention(o, sets[1][6])
        assert q27.device_status() == 0
    finally:
        torch.cuda.synchronize()
        q27.workspace_destroy()


def test_tensors_that_are_too_small_or_elsewhere(q27):
    st = H.Store([100], 6, 2, False, True, seed=1)
    kc, vc = st.new(), st.new()
    qn, qg = H.queries(st, 3)
    o = torch.zeros((6, 12, H.AD), dtype=torch.float16, device="cuda")
    mask = torch.zeros(6, dtype=torch.int64, device="cuda")
    good = [qn, qg, kc, vc, o, None, None, st.pos0, mask]
    nums = (6, H.SCALE, 12, 2, st.n_ctx)
    for i, name in ((0, "elements"), (1, "elements"), (2, "bytes"), (3, "bytes"), (4, "elements"), (8, "elements")):
        bad = list(good)
        bad[i] = good[i].flatten()[:-16 if i != 8 else -1]
        with pytest.raises(q27.Q27Error, match="expected at least .* " + name):
            q27.attn_decode_tree(*bad, *nums)
    for i, other in ((0, qn.half()), (4, o.float()), (7, st.pos0.long()), (8, mask.int())):
        bad = list(good)
        bad[i] = other
        with pytest.raises(q27.Q27Error, match="expected dtype"):
            q27.attn_decode_tree(*bad, *nums)
    bad = list(good)
    bad[0] = torch.zeros(qn.numel() + 1, device="cuda")[1:]
    with pytest.raises(q27.Q27Error, match="16-byte aligned"):
        q27.attn_decode_tree(*bad, *nums)
    with pytest.raises(q27.Q27Error, match="contiguous"):
        q27.attn_decode_tree(qn.expand(2, 6, 12, H.AD), *good[1:], *nums)


@pytest.mark.parametrize("mode", ["0", "1"])
def test_other_launch_modes(q27, mode):
    """Without programmatic launches, and with every kernel launched that way."""
    import os
    import subprocess
    import sys

    from conftest import ROOT
    subset = ["tests/test_gpu_tree.py::test_against_64_bits", "tests/test_gpu_tree.py::test_replayed_graph_sees_new_positions_and_masks",
              "tests/test_gpu_blocks.py::test_a_speculative_step", "tests/test_gpu_blocks.py::test_all_blocks_are_attn_decode",
              "tests/test_gpu_blocks.py::test_blocks_against_64_bits"]
    r = subprocess.run([sys.executable, "-m", "pytest", "-x", "-q", "-m", "gpu", "-p", "no:cacheprovider"] + subset, cwd=ROOT,
                       env=dict(os.environ, Q27_PDL=mode), capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stdout[-3000:] + r.stderr[-1000:]
    assert " passed" in r.stdout


@pytest.mark.parametrize("q8", [True, False])
@pytest.mark.parametrize("nkvh", [1, 4])
@pytest.mark.parametrize("T", [1, 2, 3, 4])
def test_few_drafts(q27, T, nkvh, q8):
    """Up to four drafts of one sequence, with a prefix of nothing, up to and past a tile, and of many parts; in a cache that ends
    there and in a long one (an f16 cache of more than 32,768 rows takes the kernel of wide trees)."""
    for n in (T, T + 1, T + 63, T + 64, T + 65, 700, 9001):
        for n_ctx in (n, 40000):
            st = H.Store([n], T, nkvh, False, q8, seed=n, n_ctx=n_ctx)
            kc, vc = st.new(), st.new()
            st.fill(kc, H.gen(n))
            st.fill(vc, H.gen(n + 1))
            masks = H.random_masks(1, T, seed=n)
            if n == 700:
                masks[0][T - 1] = 0  # sees the prefix alone
            qn, qg = H.queries(st, 3)
            o = H.call_tree(q27, st, kc, vc, qn, qg, H.mask_tensor(masks))
            H.check_attention(o, H.attention(st, kc, vc, qn, qg, H.tree_visible(st, masks)))
    assert q27.device_status() == 0


@pytest.mark.parametrize("T", [1, 2, 3, 4])
@pytest.mark.parametrize("lens", [[4], [5, 300, 128, 132], [1000] * 9 + [64] * 5, [100, 9000], [4100, 700] * 20])
def test_few_drafts_of_a_batch(q27, lens, T):
    st = H.Store(lens, T, 2, True, True, seed=T)
    kc, vc = st.new(), st.new()
    st.fill(kc, H.gen(1))
    st.fill(vc, H.gen(2))
    masks = H.random_masks(st.B, T, seed=T)
    qn, qg = H.queries(st, 3)
    o = H.call_tree(q27, st, kc, vc, qn, qg, H.mask_tensor(masks))
    H.check_attention(o, H.attention(st, kc, vc, qn, qg, H.tree_visible(st, masks)))
    assert torch.equal(o, H.call_tree(q27, st, kc, vc, qn, qg, H.mask_tensor(masks)))
    assert q27.device_status() == 0


@pytest.mark.parametrize("paged,q8", [(False, True), (False, False), (True, True)])
def test_few_drafts_poisoned_rows_and_runaway_scores(q27, paged, q8):
    """Drafts that nobody sees are NaN, beside the last rows of the prefix in their tile; the scores of those that are seen are
    far above or below those of the prefix (tolerance as for scores that run away)."""
    T, lens = 4, [333, 68, 4] if paged else [333]
    st = H.Store(lens, T, 2, paged, q8, seed=4)
    kc, vc = st.new(), st.new()
    st.fill(kc, H.gen(1))
    st.fill(vc, H.gen(2))
    qn, qg = H.queries(st, 3)
    for b, n in enumerate(lens):
        for h in range(2):
            st.poison(kc, b, h, [n - 3, n - 1])
            st.poison(vc, b, h, [n - 3, n - 1])
            st.write(kc, b, h, [n - 4, n - 2], 40.0 * torch.cat([qn[b, 0, 6 * h][None], -qn[b, 2, 6 * h][None]]))
    masks = [[0b0001, 0b0001, 0b0101, 0b0100] for _ in lens]
    o = H.call_tree(q27, st, kc, vc, qn, qg, H.mask_tensor(masks))
    ref = H.attention(st, kc, vc, qn, qg, H.tree_visible(st, masks))
    ds = ref[2] * (2.0 ** -10 + 2.0 ** -16)
    tol = ref[1] * (torch.expm1(2 * ds) + 2.0 ** -10)[..., None] + (ref[3] * 2.0 ** -25)[..., None] + ref[0].abs() * 2.0 ** -11 + 2.0 ** -25
    assert ((o.view(ref[0].shape).double() - ref[0]).abs() <= tol).all()
    assert q27.device_status() == 0


@pytest.mark.parametrize("paged,q8", [(False, True), (False, False), (True, True)])
def test_few_drafts_that_see_what_is_not_finite(q27, paged, q8):
    T, n = 4, 390
    st = H.Store([n], T, 2, paged, q8, seed=3)
    kc, vc = st.new(), st.new()
    st.fill(kc, H.gen(1))
    st.fill(vc, H.gen(2))
    mask = H.mask_tensor([[0b0001, 0b0010, 0b0111, 0b1000]])
    qn, qg = H.queries(st, 3)
    clean = H.call_tree(q27, st, kc, vc, qn, qg, mask)[0]
    for which in ("k", "v"):
        k2, v2 = kc.clone(), vc.clone()
        for h in range(2):
            st.poison(k2 if which == "k" else v2, 0, h, [n - T])
        o = H.call_tree(q27, st, k2, v2, qn, qg, mask)[0]
        for t in range(T):
            assert torch.isnan(o[t]).all() if t in (0, 2) else torch.equal(o[t], clean[t]), (which, t)


def test_few_drafts_no_length_and_bad_pages(q27):
    """Sequences shorter than their drafts, of no length, of a negative one; page indices outside the pool are reported, and the other
    sequences keep their results."""
    T = 4
    st = H.Store([0, 3, 300, 4, 700], T, 2, True, True, seed=2)
    kc, vc = st.new(), st.new()
    st.fill(kc, H.gen(1))
    st.fill(vc, H.gen(2))
    masks = [[0b1111, 0b0011, 0b1100, 0b1000]] * 5
    qn, qg = H.queries(st, 3)
    mask = H.mask_tensor(masks)
    o = H.call_tree(q27, st, kc, vc, qn, qg, mask)
    assert (o[0] == 0).all()
    H.check_attention(o, H.attention(st, kc, vc, qn, qg, H.tree_visible(st, masks)))
    st.seq_len[0] = -7
    assert torch.equal(H.call_tree(q27, st, kc, vc, qn, qg, mask), o)
    assert q27.device_status() == 0
    for seq, page in ((4, 0), (4, 2), (2, 1)):  # in the prefix, and under the drafts (positions 696 .. and 296 ..)
        good = st.table[seq, page].item()
        for bad in (-5, st.n_pages, 2 ** 31 - 1):
            st.table[seq, page] = bad
            got = H.call_tree(q27, st, kc, vc, qn, qg, mask)
            assert q27.device_status() == 2
            assert all(torch.equal(got[b], o[b]) for b in range(5) if b != seq)
        st.table[seq, page] = good
    assert torch.equal(H.call_tree(q27, st, kc, vc, qn, qg, mask), o)


@pytest.mark.parametrize("q8", [True, False])
def test_few_drafts_replayed_on_another_stream(q27, q8):
    """A captured call sees new positions and masks, with the query still being written before it; f16 and q8_1 output."""
    T, nkvh = 3, 4
    st = H.Store([1500], T, nkvh, False, q8, seed=4)
    kc, vc = st.new(), st.new()
    st.fill(kc, H.gen(1))
    st.fill(vc, H.gen(2))
    qn, qg = H.queries(st, 3)
    mask = H.mask_tensor(H.random_masks(1, T, seed=1))
    o = torch.zeros((1, T, st.nqh, H.AD), dtype=torch.float16, device="cuda")
    xq, xd = torch.zeros(o.shape, dtype=torch.int8, device="cuda"), torch.zeros(o.numel() // 32, device="cuda")
    qn2 = torch.zeros_like(qn)

    def step():
        qn2.zero_()
        for _ in range(10):
            qn2.add_(qn, alpha=0.05)
        qn2.copy_(qn)
        H.call_tree(q27, st, kc, vc, qn2, qg, mask, o)
        H.call_tree(q27, st, kc, vc, qn2, qg, mask, None, xq, xd)

    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for n, seed in ((1500, 1), (T, 2), (64, 3), (T + 1, 4), (777, 5)):
        masks = H.random_masks(1, T, seed=seed)
        st.lens = [n]
        st.pos0.fill_(n - T)
        mask.copy_(H.mask_tensor(masks))
        graph.replay()
        H.check_attention(o, H.attention(st, kc, vc, qn, qg, H.tree_visible(st, masks)))
        d, ob = xd.view(-1, 1).double(), o.view(-1, 32).double()
        assert ((xq.view(-1, 32).double() * d - ob).abs() <= d * 0.501 + ob.abs() * 2.0 ** -10 + 1e-7).all()


@pytest.mark.parametrize("mode", ["0", "1"])
def test_few_drafts_in_other_launch_modes(q27, mode):
    import os
    import subprocess
    import sys

    from conftest import ROOT
    subset = ["tests/test_gpu_tree.py::test_few_drafts_of_a_batch", "tests/test_gpu_tree.py::test_few_drafts_replayed_on_another_stream"]
    r = subprocess.run([sys.executable, "-m", "pytest", "-x", "-q", "-m", "gpu", "-p", "no:cacheprovider"] + subset, cwd=ROOT,
                       env=dict(os.environ, Q27_PDL=mode), capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stdout[-3000:] + r.stderr[-1000:]
    assert " passed" in r.stdout
