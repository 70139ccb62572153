"""Trees of drafts and chosen blocks where they can go wrong: single values that are not finite, pages that do not exist, lists and
parts of every length, lengths behind the bound that the caller gives, scores that cancel."""
import math
import random

import pytest
import torch

import helpers_rows as H

pytestmark = pytest.mark.gpu

FORMS = [(False, True, None), (False, False, None), (False, False, 40000), (True, True, None)]  # paged, q8, n_ctx


def close(o, ref, where):
    """As H.check_attention, value by value, where `where` is set; the norm there as well."""
    y, absy, amax, inv = ref
    ds = amax * (2.0 ** -10 + 2.0 ** -16)
    tol = absy * (torch.expm1(2 * ds) + 2.0 ** -10 + 2.0 ** -18)[..., None] + (inv * 2.0 ** -25)[..., None] + y.abs() * 2.0 ** -11 + 2.0 ** -25
    d = (o.view(y.shape).double() - y).abs()[where]
    assert torch.isfinite(d).all()
    assert (d <= tol[where]).all(), (d - tol[where]).max()
    assert d.norm() <= 2.0 ** -9 * y[where].norm() + 1e-6


# ---------------------------------------------------------------- values that are not finite
@pytest.mark.parametrize("paged,q8,n_ctx", FORMS)
@pytest.mark.parametrize("T", [2, 4, 5, 11, 33])
def test_one_infinite_value_stays_in_its_dim(q27, T, paged, q8, n_ctx):
    """Single values of drafted V rows: infinities and NaN of an f16 row; of a q8_0 row a NaN scale (32 dims), and a value whose
    product with its scale, 127 * 600 = 76,200, f16 does not hold although the result is finite. The other dims, and the drafts that do not
    see these rows, are what they are without; NaN and infinities come out where the formula has them (no weight underflows here)."""
    n = 300
    st = H.Store([n] if not paged else [n, 70 + T], T, 2, paged, q8, seed=3, n_ctx=n_ctx)
    kc, vc = st.new(), st.new()
    st.fill(kc, H.gen(1))
    st.fill(vc, H.gen(2))
    clean = vc.clone()
    v, s = st.parts(vc)
    for b, ln in enumerate(st.lens):
        for h in range(2):
            rows = [int(st.index(b, h, [ln - T + j])) for j in (0, 1, T - 1)]
            if s is None:
                v[rows[0], 37], v[rows[0], 200] = math.inf, -math.inf
                v[rows[1], 41] = math.nan
                v[rows[2], 200] = math.inf
            else:
                v[rows[0], 32:64], s[rows[0], 1] = 0, 600.0
                v[rows[0], 37], v[rows[0], 41] = 127, -2
                s[rows[1], 3] = math.nan
                v[rows[2], 224:256], s[rows[2], 7] = 0, 600.0
                v[rows[2], 255] = -120
    masks = [[(1 << t) | (0b11 if t % 3 == 0 else 0) | (1 << (T - 1) if t % 2 else 0) for t in range(T)] for _ in st.lens]
    if T > 2:
        masks = [[m if t != 2 else 1 << 2 for t, m in enumerate(row)] for row in masks]
    qn, qg = H.queries(st, 3)
    ref = H.attention(st, kc, vc, qn, qg, H.tree_visible(st, masks))
    inv = H.attention(st, kc, clean, qn, qg, H.tree_visible(st, masks))[3]  # (P in f16 meets the other values only)
    o = H.call_tree(q27, st, kc, vc, qn, qg, H.mask_tensor(masks)).view(ref[0].shape)
    y = ref[0]
    assert not torch.isfinite(y).all() and (T < 4 or torch.isfinite(y[:, 2]).all())
    assert torch.equal(torch.isnan(o), torch.isnan(y))
    assert torch.equal(o == math.inf, y == math.inf) and torch.equal(o == -math.inf, y == -math.inf)
    close(o, (*ref[:3], inv), torch.isfinite(y))
    assert q27.device_status() == 0


# ---------------------------------------------------------------- pages that do not exist
@pytest.mark.parametrize("T", [1, 3, 4, 5, 30])
@pytest.mark.parametrize("where", ["first", "middle", "prefix end", "drafts"])
def test_rows_of_a_page_that_does_not_exist_are_not_seen(q27, T, where):
    """Every sequence of the batch has its result: the one with the bad page that of the other pages' rows alone."""
    lens = [1100, 300 + T, 2000]
    st = H.Store(lens, T, 2, True, True, seed=T)
    kc, vc = st.new(), st.new()
    st.fill(kc, H.gen(1))
    st.fill(vc, H.gen(2))
    masks = H.random_masks(3, T, seed=T)
    qn, qg = H.queries(st, 3)
    b = 2
    page = {"first": 0, "middle": 3, "prefix end": (lens[b] - T - 1) // 256, "drafts": (lens[b] - 1) // 256}[where]
    whole = H.tree_visible(st, masks)
    ref = H.attention(st, kc, vc, qn, qg, lambda s, t, h: [p for p in whole(s, t, h) if s != b or p // 256 != page])
    for bad in (-1, st.n_pages, 2 ** 31 - 1, -2 ** 31):
        st.table[b, page] = bad
        o = H.call_tree(q27, st, kc, vc, qn, qg, H.mask_tensor(masks))
        assert q27.device_status() == 2
        H.check_attention(o, ref)


def test_no_page_at_all(q27):
    for T in (2, 7):
        st = H.Store([700], T, 2, True, True, seed=T)
        kc, vc = st.new(), st.new()
        st.fill(kc, H.gen(1))
        st.fill(vc, H.gen(2))
        st.table.fill_(-1)
        qn, qg = H.queries(st, 3)
        o = H.call_tree(q27, st, kc, vc, qn, qg, H.mask_tensor(H.random_masks(1, T, seed=1)))
        assert (o == 0).all() and q27.device_status() == 2


@pytest.mark.parametrize("page", [0, 2, 7])
def test_blocks_of_a_page_that_does_not_exist_are_not_seen(q27, page):
    lens, T, k = [2000, 500], 2, 12
    st = H.Store(lens, T, 2, True, True, seed=1)
    kc, vc = st.new(), st.new()
    st.fill(kc, H.gen(1))
    st.fill(vc, H.gen(2))
    qn, qg = H.queries(st, 3)
    r = random.Random(page)
    sel = torch.tensor([[[sorted(r.sample(range(-(-n // 64)), min(k, -(-n // 64)))) + [-1] * (k - min(k, -(-n // 64))) for _ in range(2)]
                         for _ in range(T)] for n in lens], dtype=torch.int32)
    sel[0, :, :, 0] = 4 * page

    def visible(b, t, h):
        last = lens[b] - T + t
        return [p for x in sel[b, t, h].tolist() if x >= 0 and not (b == 0 and x // 4 == page) for p in range(64 * x, min(64 * x + 64, last + 1))]
    ref = H.attention(st, kc, vc, qn, qg, visible)
    st.table[0, page] = st.n_pages
    o = H.call_blocks(q27, st, kc, vc, qn, qg, sel.cuda())
    assert q27.device_status() == 2
    H.check_attention(o, ref)


# ---------------------------------------------------------------- workspace
def test_the_query_counts_outgrown_buffers_and_a_fixed_size_is_exact(q27):
    def step(lens, T):
        st = H.Store(lens, T, 2, True, True, seed=1)
        kc, vc = st.new(), st.new()
        st.fill(kc, H.gen(1))
        st.fill(vc, H.gen(2))
        masks = H.random_masks(st.B, T, seed=1)
        qn, qg = H.queries(st, 3)
        o = H.call_tree(q27, st, kc, vc, qn, qg, H.mask_tensor(masks))
        H.check_attention(o, H.attention(st, kc, vc, qn, qg, H.tree_visible(st, masks)))
    try:
        q27.workspace_destroy()
        step([200], 2)
        first = q27.workspace_query()[2]
        step([200] * 3, 9)
        both = q27.workspace_query()[2]
        live = both - first
        assert first > 0 and live >= first + first // 2
        q27.workspace_init(0, live + 4096)
        assert q27.workspace_query()[2:] == (both + live + 4096, True)
        step([200] * 3, 9)
    finally:
        torch.cuda.synchronize()
        q27.workspace_destroy()
    assert q27.workspace_query() == (0, 0, 0, False)


# ---------------------------------------------------------------- every size of the kernels
def reference_bounds(st, kc, bounds, T):
    want = bounds.clone()
    for b, n in enumerate(st.lens):
        lo, nb = max(0, n - T) // 64, -(-n // 64)
        if n - T >= n or n <= 0:
            continue
        for h in range(st.nkvh):
            x = st.read(kc, b, h, range(64 * lo, n)).half()
            at = torch.tensor([H.bounds_at(st, b, h, i) for i in range(lo, nb)], device="cuda")
            pad = torch.cat([x, x[-1:].expand(64 * (nb - lo) - len(x), -1)]).view(nb - lo, 64, H.AD)
            want[at, 0], want[at, 1] = pad.amin(1), pad.amax(1)
    return want


@pytest.mark.parametrize("lens,T,nkvh,paged", [
    ([64 * 460 + 17], 64 * 460 + 17, 4, False), ([64 * 520 + 63], 64 * 470 + 5, 4, False), ([64 * 1900 + 1], 64 * 1800, 1, False),
    ([8000, 12345, 9001, 8064], 8000, 4, True), ([9000, 100, 7001, 0, 8999, 64], 7001, 4, True)])
def test_bounds_of_many_blocks(q27, lens, T, nkvh, paged):
    """From 12 blocks for an SM on a warp takes a block; odd ends, sequences shorter than T, and rows whose scale is NaN."""
    st = H.Store(lens, T, nkvh, paged, True, seed=T)
    assert ((T + 62) // 64 + 1) * nkvh * len(lens) >= 12 * torch.cuda.get_device_properties(0).multi_processor_count
    kc = st.new()
    st.fill(kc, H.gen(1), 3.0)
    bounds = H.new_bounds(q27, st, 7.5)
    want = reference_bounds(st, kc, bounds, T)
    H.call_bounds(q27, st, kc, bounds, T)
    assert torch.equal(bounds, want)
    n = lens[0]
    st.poison(kc, 0, nkvh - 1, [n - 1, n - 64 * 70])
    H.call_bounds(q27, st, kc, bounds, T)
    bad = {H.bounds_at(st, 0, nkvh - 1, p // 64) for p in (n - 1, n - 64 * 70)}
    nan = torch.isnan(bounds).all(-1).all(-1)
    assert set(nan.nonzero().flatten().tolist()) == bad and not torch.isnan(bounds[~nan]).any()
    assert torch.equal(bounds[~nan], want[~nan])
    assert q27.device_status() == 0


@pytest.mark.parametrize("T", [1, 2, 3, 4])
def test_choice_in_a_batch_of_long_and_short_sequences(q27, T):
    """More groups of 64 blocks than a (KV head, sequence) has CTAs: each goes through several."""
    r = random.Random(T)
    lens = [T, 24000, 300 + T, 23999, 64, 16385] + [r.randrange(T, 24000) for _ in range(34)]
    st = H.Store(lens, T, 4, True, True, seed=T)
    bounds = H.new_bounds(q27, st)
    bounds.copy_(torch.randn(bounds.shape, generator=H.gen(T), device="cuda") + torch.tensor([-2.0, 2.0], device="cuda")[:, None])
    qn, _ = H.queries(st, 3)
    for k, sink, recent in ((5, 1, 2), (100, 0, 1)):
        assert torch.equal(H.call_select(q27, st, qn, bounds, k, sink, recent).cpu(), H.select_reference(st, qn, bounds, k, sink, recent))
    assert q27.device_status() == 0


def long_list(nb, k, full, r):
    """A list of k entries: `full` blocks at its front, the others anywhere behind, -1 between them, and some entries that are none."""
    blocks = r.sample(range(nb), nb)
    out = blocks[:full] + [-1] * (k - full)
    at = r.sample(range(full, k), min(k - full, nb - full) // 2 + (k - full) // 50)
    for i, x in zip(at, blocks[full:] + [-2, 2 ** 30, -2 ** 31] * k):
        out[i] = x
    return out


@pytest.mark.parametrize("paged,q8", [(False, True), (False, False), (True, True)])
@pytest.mark.parametrize("k,full,n,T", [(129, 100, 9000, 4), (1000, 200, 30000, 2), (16384, 128, 30000, 2)])
def test_lists_of_every_length(q27, paged, q8, k, full, n, T):
    """Chunks of a list up to the 128 entries that a CTA takes, whole or with blocks far behind each other."""
    lens = [n, 5000, 64 * full + T] if paged else [n]
    st = H.Store(lens, T, 2, paged, q8, seed=k)
    kc, vc = st.new(), st.new()
    st.fill(kc, H.gen(1))
    st.fill(vc, H.gen(2))
    r = random.Random(k)
    sel = torch.tensor([[[long_list((ln - T + t) // 64 + 1, k, min(full, (ln - T + t) // 64 + 1), r) for _ in range(2)] for t in range(T)]
                        for ln in lens], dtype=torch.int32)
    qn, qg = H.queries(st, 3)

    def visible(b, t, h):
        last = st.lens[b] - T + t
        return [p for x in sel[b, t, h].tolist() if 0 <= x <= last // 64 for p in range(x * 64, min((x + 1) * 64, last + 1))]
    ref = H.attention(st, kc, vc, qn, qg, visible)
    o = H.call_blocks(q27, st, kc, vc, qn, qg, sel.cuda())
    H.check_attention(o, ref)
    assert q27.device_status() == (4 if ((sel < -1) | (sel == 2 ** 30)).any() else 0)  # entries that are none
    sel[(sel < 0) | (sel > n // 64)] = -1
    assert torch.equal(H.call_blocks(q27, st, kc, vc, qn, qg, sel.cuda()), o)
    assert q27.device_status() == 0


def test_many_lists(q27):
    """Pairs of CTAs on an SM: more chunks than SMs."""
    T, k, lens = 4, 150, [4000 + 300 * i for i in range(20)]
    st = H.Store(lens, T, 4, True, True, seed=1)
    kc, vc = st.new(), st.new()
    st.fill(kc, H.gen(1))
    st.fill(vc, H.gen(2))
    r = random.Random(1)
    sel = torch.tensor([[[sorted(r.sample(range(-(-n // 64)), 50)) + [-1] * (k - 50) for _ in range(4)] for _ in range(T)] for n in lens],
                       dtype=torch.int32)
    qn, qg = H.queries(st, 3)

    def visible(b, t, h):
        last = lens[b] - T + t
        return [p for x in sel[b, t, h].tolist() if x >= 0 for p in range(x * 64, min((x + 1) * 64, last + 1))]
    H.check_attention(H.call_blocks(q27, st, kc, vc, qn, qg, sel.cuda()), H.attention(st, kc, vc, qn, qg, visible))
    assert q27.device_status() == 0


def test_long_parts_of_a_batch(q27):
    """Parts of more than 32 tiles, with and without pages that do not exist in their second half."""
    T, nkvh, lens = 6, 4, [20000, 12001, 17000, 19937, 3, 16000, 13999, 20000]
    st = H.Store(lens, T, nkvh, True, True, seed=1)
    kc, vc = st.new(), st.new()
    st.fill(kc, H.gen(1))
    st.fill(vc, H.gen(2))
    masks = H.random_masks(st.B, T, seed=2)
    qn, qg = H.queries(st, 3)
    whole = H.tree_visible(st, masks)
    H.check_attention(H.call_tree(q27, st, kc, vc, qn, qg, H.mask_tensor(masks)), H.attention(st, kc, vc, qn, qg, whole))
    assert q27.device_status() == 0
    bad = {0: {10, 22, 23, 50}, 3: {9, 77}, 6: {40}}  # sequence -> pages of four tiles
    for b, pages in bad.items():
        for pg in pages:
            st.table[b, pg] = -1
    ref = H.attention(st, kc, vc, qn, qg, lambda b, t, h: [p for p in whole(b, t, h) if p // 256 not in bad.get(b, ())])
    H.check_attention(H.call_tree(q27, st, kc, vc, qn, qg, H.mask_tensor(masks)), ref)
    assert q27.device_status() == 2


# ---------------------------------------------------------------- a bound that is not the longest length
def widen_table(st, pages):
    more = torch.full((st.B, pages - st.max_pages), -1, dtype=torch.int32, device="cuda")
    st.table, st.max_pages = torch.cat([st.table, more], 1).contiguous(), pages


@pytest.mark.parametrize("T", [1, 4, 5, 20])
@pytest.mark.parametrize("bound", [200, 700, 1003, 5000, 100000])
def test_trees_and_the_bound_of_the_lengths(q27, T, bound):
    """Sequences behind max_seq_len are cut there, drafts among what is cut; a bound far above the lengths changes nothing."""
    lens = [1000, 150, 730, T, 705]
    st = H.Store(lens, T, 2, True, True, seed=T)
    kc, vc = st.new(), st.new()
    st.fill(kc, H.gen(1))
    st.fill(vc, H.gen(2))
    widen_table(st, 400)
    st.max_len = bound
    masks = H.random_masks(st.B, T, seed=T)
    qn, qg = H.queries(st, 3)
    whole = H.tree_visible(st, masks)
    ref = H.attention(st, kc, vc, qn, qg, lambda b, t, h: [p for p in whole(b, t, h) if p < bound])
    H.check_attention(H.call_tree(q27, st, kc, vc, qn, qg, H.mask_tensor(masks)), ref)
    assert q27.device_status() == 0


@pytest.mark.parametrize("T", [1, 3])
@pytest.mark.parametrize("bound", [64, 1000, 1003, 5000, 100000])
def test_choice_and_the_bound_of_the_lengths(q27, T, bound):
    lens = [4000, 150, 1500, 64, 1010]
    st = H.Store(lens, T, 2, True, True, seed=T)
    bounds = H.new_bounds(q27, st)
    bounds.copy_(torch.randn(bounds.shape, generator=H.gen(T), device="cuda") + torch.tensor([-2.0, 2.0], device="cuda")[:, None])
    qn, _ = H.queries(st, 3)
    want = []
    for t in range(T):  # a token at position p chooses as the last token of a sequence of min(p + 1, bound) positions
        one = H.Store([min(n - T + t + 1, bound) for n in lens], 1, 2, True, True, seed=T)
        one.host_table = st.host_table
        want.append(H.select_reference(one, qn[:, t:t + 1], bounds, 6, 1, 2))
    widen_table(st, 400)
    st.max_len = bound
    assert torch.equal(H.call_select(q27, st, qn, bounds, 6, 1, 2).cpu(), torch.cat(want, 1))
    assert q27.device_status() == 0


# ---------------------------------------------------------------- scores that cancel
@pytest.mark.parametrize("T", [1, 2, 4])
@pytest.mark.parametrize("kind", ["equal", "halves", "mixed", "steps"])
def test_scores_that_cancel(q27, kind, T):
    """Scores that are tiny beside the sum A of the products' magnitudes and differ by 2^-12 to 2^-20 of it, at the resolution of the
    first pass (2^-14 A) and below: a block that its rounded score settled wrongly would show. The products are exact in 64 bits and their sums are
    off by less than 2^-43 A."""
    n_blocks, k = 700, 90
    st = H.Store([64 * n_blocks], T, 2, False, True, seed=1, n_ctx=64 * n_blocks)
    g = H.gen(T)
    rnd = lambda *s: torch.rand(s, generator=g, device="cuda")  # noqa: E731
    sign = lambda *s: torch.where(rnd(*s) < 0.5, -1.0, 1.0)  # noqa: E731
    for scale in (1.0, 2.0 ** -9, 300.0):
        bounds = H.new_bounds(q27, st, 0.0)
        N = bounds.shape[0]
        if kind == "steps":  # one vector of values, of a few of which the last bit differs; the query's signs cancel its sum
            x = (1 + rnd(H.AD)).half()
            v = x.view(torch.int16).repeat(N, 1) + (rnd(N, H.AD) < 0.3).to(torch.int16)
            v = v.view(torch.float16).float()
            a = (1 + rnd(H.AD)) * sign(H.AD)
            a[-1] = -(a[:-1] * x[:-1].float()).sum() / x[-1].float()
        else:  # the second half takes back what the first gives, but for one dim
            big = {"equal": torch.ones(N, 1, device="cuda"), "halves": 1 + rnd(N, 1), "mixed": torch.exp2(-8 * rnd(N, 1))}[kind]
            half = (big * (1 + rnd(N, 128)) * sign(N, 128)).half().float()
            v = torch.cat([half, half], 1)
            a = (1 + rnd(128)) * sign(128)
            a = torch.cat([a, -a])
            A = 2 * (a[:128].abs() * half.abs()).sum(-1).mean()
            step = 2.0 ** (-12 - 8 * torch.rand(N, generator=g, device="cuda"))
            v[:, 5] += A * step * sign(N) / a[5].abs()
        v = (v * scale).half()
        bounds[:, 0], bounds[:, 1] = v, v  # (lo = hi: the score is q.v)
        qn = a.repeat(1, T, st.nqh, 1) * torch.exp2(torch.arange(T * st.nqh, device="cuda") % 5 - 2.0).view(1, T, st.nqh, 1)
        assert torch.equal(H.call_select(q27, st, qn, bounds, k, 1, 2).cpu(), H.select_reference(st, qn, bounds, k, 1, 2)), scale
    assert q27.device_status() == 0


# ---------------------------------------------------------------- shapes and positions at the ends of what is allowed
@pytest.mark.parametrize("T", [2, 5])
def test_more_sequences_than_threads(q27, T):
    r = random.Random(T)
    lens = [r.choice([0, 1, T, 64, 70]) for _ in range(1300)]
    st = H.Store(lens, T, 1, True, True, seed=T)
    kc, vc = st.new(), st.new()
    g = H.gen(1)
    for buf in (kc, vc):
        v, s = st.parts(buf)
        v.copy_(torch.randint(-127, 128, v.shape, generator=g, device="cuda", dtype=torch.int8))
        s.copy_(torch.rand(s.shape, generator=g, device="cuda") * 0.02)
    masks = H.random_masks(st.B, T, seed=T)
    qn, qg = H.queries(st, 3)
    o = H.call_tree(q27, st, kc, vc, qn, qg, H.mask_tensor(masks))
    H.check_attention(o, H.attention(st, kc, vc, qn, qg, H.tree_visible(st, masks)))
    assert q27.device_status() == 0


@pytest.mark.parametrize("nkvh,n_ctx", [(7, 131), (16, 200), (149, 70), (200, 65)])
@pytest.mark.parametrize("q8", [True, False])
def test_many_heads(q27, nkvh, n_ctx, q8):
    """More KV heads than SMs among them: trees, their commit, bounds, choice and lists."""
    for T in (2, 6):
        n = n_ctx - 3
        st = H.Store([n], T, nkvh, False, q8, seed=T, n_ctx=n_ctx)
        kc, vc = st.new(), st.new()
        st.fill(kc, H.gen(1))
        st.fill(vc, H.gen(2))
        masks = H.random_masks(1, T, seed=T)
        qn, qg = H.queries(st, 3)
        o = H.call_tree(q27, st, kc, vc, qn, qg, H.mask_tensor(masks))
        H.check_attention(o, H.attention(st, kc, vc, qn, qg, H.tree_visible(st, masks)))
        if T == 2:
            bounds = H.new_bounds(q27, st, 7.5)
            want = reference_bounds(st, kc, bounds, n)
            H.call_bounds(q27, st, kc, bounds, n)
            assert torch.equal(bounds, want)
            sel = H.call_select(q27, st, qn, bounds, 2, 0, 1)
            ref = H.select_reference(st, qn, bounds, 2, 0, 1)
            assert torch.equal(sel.cpu(), ref)
            seen = lambda b, t, h: [p for x in ref[b, t, h].tolist() if x >= 0 for p in range(64 * x, min(64 * x + 64, n - T + t + 1))]  # noqa: E731
            H.check_attention(H.call_blocks(q27, st, kc, vc, qn, qg, sel), H.attention(st, kc, vc, qn, qg, seen))
        k0, v0 = kc.clone(), vc.clone()
        q27.kv_commit(kc, vc, st.pos0, H.i32([T - 1] + [0] * (T - 1)), H.i32([1]), T, nkvh, n_ctx, q8)
        for new, old in ((kc, k0), (vc, v0)):
            (a, sa), (b, sb) = st.parts(new), st.parts(old)
            at = torch.tensor([int(st.index(0, h, [n - T])) for h in range(nkvh)], device="cuda")
            b[at] = b[at + T - 1]
            if sb is not None:
                sb[at] = sb[at + T - 1]
            assert torch.equal(new, old)
    assert q27.device_status() == 0


@pytest.mark.parametrize("q8", [True, False])
@pytest.mark.parametrize("T", [3, 9])
def test_drafts_outside_the_cache(q27, T, q8):
    """Positions before the cache and behind it: what lies inside is attended, the rest is not there."""
    n_ctx = 150
    for pos in (-T, 1 - T, -1, n_ctx - T, n_ctx - T + 1, n_ctx - 1, n_ctx, n_ctx + 70):
        st = H.Store([n_ctx], T, 2, False, q8, seed=T, n_ctx=n_ctx)
        kc, vc = st.new(), st.new()
        st.fill(kc, H.gen(1))
        st.fill(vc, H.gen(2))
        masks = H.random_masks(1, T, seed=T, empty=False)
        qn, qg = H.queries(st, 3)
        st.pos0.fill_(pos)

        def seen(b, t, h):
            return [p for p in range(n_ctx) if p < pos] + [pos + j for j in range(T) if 0 <= pos + j < n_ctx and (masks[0][t] >> j) & 1]
        o = H.call_tree(q27, st, kc, vc, qn, qg, H.mask_tensor(masks))
        H.check_attention(o, H.attention(st, kc, vc, qn, qg, seen))
        if T == 3:
            sel = torch.arange(3, dtype=torch.int32, device="cuda").expand(1, T, 2, 3).contiguous()
            o = H.call_blocks(q27, st, kc, vc, qn, qg, sel)
            H.check_attention(o, H.attention(st, kc, vc, qn, qg, lambda b, t, h: list(range(max(0, min(n_ctx, pos + t + 1))))))
            bounds = H.new_bounds(q27, st, 0.0)
            got = H.call_select(q27, st, qn, bounds, 4, 1, 1)[0, :, 0].tolist()
            nb = [max(0, min(n_ctx - 1, pos + t) // 64 + 1) if pos + t >= 0 else 0 for t in range(T)]
            assert got == [list(range(x)) + [-1] * (4 - x) for x in nb]
    assert q27.device_status() == 0


@pytest.mark.parametrize("paged,q8,n_ctx", FORMS)
@pytest.mark.parametrize("T", [4, 7])
def test_a_query_that_is_not_finite_stays_in_its_row(q27, T, paged, q8, n_ctx):
    st = H.Store([500], T, 2, paged, q8, seed=T, n_ctx=n_ctx)
    kc, vc = st.new(), st.new()
    st.fill(kc, H.gen(1))
    st.fill(vc, H.gen(2))
    masks = H.random_masks(1, T, seed=T)
    qn, qg = H.queries(st, 3)
    clean = H.call_tree(q27, st, kc, vc, qn, qg, H.mask_tensor(masks))
    qn[0, 1, 3, 17], qn[0, 2, 8, 200] = math.nan, math.inf
    o = H.call_tree(q27, st, kc, vc, qn, qg, H.mask_tensor(masks))
    rows = torch.ones(o.shape[:3], dtype=torch.bool, device="cuda")
    rows[0, 1, 3] = rows[0, 2, 8] = False
    assert torch.isnan(o[0, 1, 3]).all() and torch.equal(o[rows], clean[rows])
    assert q27.device_status() == 0


def test_bookkeeping_over_pages_that_do_not_exist(q27):
    """Commit leaves rows whose source or destination is on no page, bounds leave such blocks, the choice ranks them last."""
    T, nkvh, lens = 6, 2, [600, 515, 3000]
    st = H.Store(lens, T, nkvh, True, True, seed=1)
    kc, vc = st.new(), st.new()
    st.fill(kc, H.gen(1))
    st.fill(vc, H.gen(2))
    good = st.table.clone()
    st.table[1, 2] = st.n_pages  # positions 512 .. of the second sequence: drafts 509 .. 514
    before = kc.clone(), vc.clone()
    path = [[5, 4, 3, 2, 1, 0]] * 3
    q27.kv_commit_paged(kc, vc, st.table, st.seq_len, H.i32(path), H.i32([6, 6, 0]), 3, T, nkvh, st.n_pages, st.max_pages)
    assert q27.device_status() == 2
    st.table.copy_(good)
    for new, old in zip((kc, vc), before):
        for h in range(nkvh):
            assert torch.equal(st.read(new, 0, h, range(594, 600)), st.read(old, 0, h, range(594, 600)).flip(0))
            assert torch.equal(st.read(new, 1, h, range(515)), st.read(old, 1, h, range(515)))
            assert torch.equal(st.read(new, 2, h, range(3000)), st.read(old, 2, h, range(3000)))
    bounds = H.new_bounds(q27, st, 7.5)
    want = reference_bounds(st, kc, bounds, 600)
    bad = {0: [1], 1: [2], 2: [10, 11]}
    for b, pages in bad.items():
        for pg in pages:
            st.table[b, pg] = -3
            for h in range(nkvh):
                for blk in range(4 * pg, 4 * pg + 4):
                    want[H.bounds_at(st, b, h, blk)] = 7.5
    H.call_bounds(q27, st, kc, bounds, 600)
    assert q27.device_status() == 2 and torch.equal(bounds, want)
    # the choice: every key is small, what the bad pages' bounds say (7.5) would win
    H.call_bounds(q27, st, kc, bounds, 3000)
    q27.device_status()
    st.T, one = 1, H.Store(lens, 1, nkvh, True, True, seed=1)
    qn, _ = H.queries(one, 3)
    sel = H.call_select(q27, st, qn, bounds, 8, 0, 1)
    assert q27.device_status() == 2
    for b, n in enumerate(lens):
        nb = (n - 1) // 64 + 1
        for h in range(nkvh):
            got = [x for x in sel[b, 0, h].tolist() if x >= 0]
            gone = [x for x in range(nb - 1) if x // 4 in bad[b]]
            assert got == sorted(got) and len(got) == min(8, nb) and got[-1] == nb - 1
            there = nb - len(gone)
            assert len([x for x in got if x in gone]) == max(0, min(8, nb) - there)
