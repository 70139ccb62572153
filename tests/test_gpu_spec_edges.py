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
