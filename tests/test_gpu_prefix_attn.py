"""b200_prefix_attn against its definition in 64 bits.

The bound: weights enter the second product rounded to the cache's type (half a step of each), the result is rounded once more; scores are F32 sums of d
products (each within d 2^-24 of the sum of magnitudes, which a weight feels as a relative error), exponentials are good to 2^-21.  A weight below the
type's normal numbers is off by SMALLEST at most, of weights whose largest is 1.  So
    |got - o| <= (half + 2 e) sum w |v| + half |o| + n SMALLEST max |v| / z + SMALLEST,     e = d 2^-24 max sum |q k| scale + 2^-21 (1 + max |score|)."""
import importlib

import numpy as np
import pytest

import b200
import plain_paged as P

pytestmark = pytest.mark.gpu
GUARD = 64


@pytest.fixture(scope="module")
def p():
    b200.load()
    return importlib.import_module("llama_rust_b200.paged")


def device(a):
    return b200.load().device_array(a)


class Problem:
    def __init__(self, p, groups, lens, shared, ty="F16", d=128, kv=2, each=2, page=16, table_pages=None, sinks=False, seed=0, scale=None, dev=1.0, table_of=None):
        """groups: sequences of each; lens, shared: by sequence"""
        rng = np.random.default_rng(seed)
        self.p, self.ty, self.d, self.kv, self.heads, self.page, self.n = p, ty, d, kv, kv * each, page, len(lens)
        self.lens, self.shared = list(lens), list(shared)
        self.first = [0] + list(np.cumsum(groups)) if groups else []
        self.pages_each = table_pages or max(1, -(-max(max(lens), 1) // page))
        self.n_pages = self.n * self.pages_each + 1
        self.tables = rng.permutation(self.n_pages)[: self.n * self.pages_each].reshape(self.n, self.pages_each).astype(np.int32)
        self.k, self.v = (P.rounded(rng.standard_normal((self.n_pages, page, kv, d)) * f, ty) for f in (dev, 1.0))
        self.q = P.rounded(rng.standard_normal((self.n, self.heads, d)) * 1.5, ty)
        self.sinks = rng.standard_normal(self.heads).astype(np.float32) if sinks else None
        self.scale = d ** -0.5 if scale is None else scale

    def call(self, hints=True, workspace=None):
        p, TY = self.p, {"F16": self.p.F16, "BF16": self.p.BF16}
        self.keep = [device(P.bits(self.k, self.ty)), device(P.bits(self.v, self.ty)), device(self.tables), device(P.bits(self.q, self.ty)),
                     device(P.bits(np.full(self.q.size + GUARD, -7.0), self.ty)), device(np.array(self.lens, dtype=np.int32)), device(np.array(self.shared, dtype=np.int32)),
                     device(np.array(self.first or [0], dtype=np.int32)), device(self.sinks if self.sinks is not None else np.zeros(1, dtype=np.float32))]
        k, v, tables, q, self.out, lens, shared, first, sinks = self.keep
        cache = p.Cache(TY[self.ty], self.page, self.n_pages, self.kv, self.d, k.ptr, v.ptr, tables.ptr, self.pages_each, self.n)
        sizes = dict(max_len=max(max(self.lens), 0), max_shared=max(max(self.shared), 0), max_group=int(np.diff(self.first).max()) if self.first else 0) if hints is True else dict(hints or {})
        return p.PrefixAttn(cache, self.n, self.heads, q.ptr, self.out.ptr, lens.ptr, self.scale, shared=shared.ptr if self.first else None, group_first=first.ptr if self.first else None,
                            n_group=max(len(self.first) - 1, 0), sinks=sinks.ptr if self.sinks is not None else None, workspace=workspace, **sizes)

    def result(self):
        got = P.values(self.out.download(np.uint16, self.q.size + GUARD), self.ty)
        assert (got[self.q.size:] == -7.0).all()
        return got[: self.q.size].reshape(self.q.shape)

    def want(self):
        with np.errstate(invalid="ignore"):
            return P.attention(self.k, self.v, self.tables.tolist(), self.q, self.lens, self.shared if self.first else [0] * self.n, self.first, self.scale, self.sinks)

    def check(self, got, error=0):
        want, size, big, total = self.want()
        fine = np.isfinite(self.k).all() and np.isfinite(self.q).all()
        top = (np.abs(self.q).max() * np.abs(self.k).max() if fine else 0.0) * abs(self.scale)
        mags = np.abs(self.q).sum(2).max() * np.abs(self.k).max() * abs(self.scale) if fine else 0.0
        # sum |q k| and |score| bounded by sum |q| max |k|
        e = self.d * 2.0 ** -24 * mags + 2.0 ** -21 * (1 + mags)
        assert top <= mags + 1e-9 or not fine
        half, small = P.HALF_STEP[self.ty], P.SMALLEST[self.ty]
        n = max(max(self.lens), 1)
        tol = (half + 2 * e) * size + half * np.abs(want) + n * small * big / total + small
        assert np.array_equal(np.isnan(got), np.isnan(want))
        with np.errstate(invalid="ignore"):
            ok = (np.abs(got - want) <= tol) | (got == want) | np.isnan(want)
        assert ok.all(), ("worst", np.nanmax(np.abs(got - want) / tol), np.argwhere(~ok)[:4])
        assert b200.load().kernel_error() == error

    def run(self, hints=True, error=0):
        self.call(hints)(None)
        self.check(self.result(), error)
        return self


@pytest.mark.parametrize("ty", ["F16", "BF16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("page", [16, 64])
def test_types_heads_and_pages(p, ty, d, page):
    Problem(p, [3, 2], [140, 133, 129, 77, 90], [128, 128, 128, 64, 64], ty, d, page=page).run()


@pytest.mark.parametrize("kv,each", [(1, 1), (1, 7), (2, 16), (1, 40), (8, 4), (3, 5), (16, 1)])
@pytest.mark.parametrize("groups,shared", [([6], 100), ([], 0)])
def test_head_layouts(p, kv, each, groups, shared):
    Problem(p, groups, [110, 100, 104, 101, 117, 133], [shared] * 6, "BF16", 64, kv, each).run()


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("shared", [1, 15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 256, 257])
def test_shared_parts_that_end_anywhere(p, page, shared):
    Problem(p, [4], [shared + 1, shared, shared + 40, shared + 129], [shared] * 4, "F16", 64, 1, 2, page).run()


@pytest.mark.parametrize("lens", [[1], [2, 1], [0, 0], [0, 1, 17, 0, 64], [65, 0]])
@pytest.mark.parametrize("groups", [True, False])
def test_shortest_lengths_and_empty_rows(p, lens, groups):
    pr = Problem(p, [len(lens)] if groups else [], lens, [1] * len(lens), sinks=True).run()
    for s, n in enumerate(lens):
        assert n > 0 or not pr.result()[s].any()


def test_rows_end_before_the_shared_part_does(p):
    Problem(p, [5, 3], [300, 10, 0, 200, 257, 1, 0, 99], [256] * 5 + [64] * 3).run()


def test_sequences_of_a_group_may_share_less(p):
    Problem(p, [5], [300, 280, 290, 100, 270], [256, 64, 0, 100, 300]).run()


def test_group_sizes(p):
    Problem(p, [1, 70, 1, 9], [150] * 81, [130] * 81, "BF16", 64, 1, 3).run()
    Problem(p, [0, 2, 1], [150] * 3, [130] * 3, "BF16", 64, 1, 3).run()


@pytest.mark.parametrize("ty,d,each", [("BF16", 128, 4), ("F16", 128, 1), ("F16", 64, 4), ("BF16", 64, 8)])
def test_many_rows_over_a_long_prefix(p, ty, d, each):
    n, shared = 40, 3000
    Problem(p, [n], [shared + (i * 13) % 200 for i in range(n)], [shared] * n, ty, d, 2, each, 32, sinks=True).run()


@pytest.mark.parametrize("each,n", [(4, 32), (4, 33), (2, 128), (1, 129), (16, 17), (40, 7)])
def test_row_blocks_that_are_not_whole(p, each, n):
    Problem(p, [n, 2], [400 + i % 50 for i in range(n + 2)], [390] * (n + 2), "BF16", 128, 1, each, 64).run()


@pytest.mark.parametrize("rows", [31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257])
@pytest.mark.parametrize("ty,d", [("F16", 64), ("BF16", 128)])
def test_blocks_of_every_kind_at_their_borders(p, rows, ty, d):
    # every form of the shared part (32, 64, 128, 256 rows a block) full, one short and one over; several tiles, rows that see fewer
    lens = [540 - (i % 5) * 128 for i in range(rows)]
    Problem(p, [rows], lens, [520] * rows, ty, d, 1, 1, 32, seed=rows).run()


@pytest.mark.parametrize("n,each", [(8, 4), (16, 4), (30, 4), (60, 4)])
def test_scores_that_grow_along_the_positions(p, n, each):
    # the maximum in use falls behind again and again: by little, by more than 2^12, and all at once
    for dev in (0.02, 0.3, 4.0):
        pr = Problem(p, [n], [900] * n, [896] * n, "BF16", 64, 1, each, 128)
        page, place = np.array([P.cell(pr.tables.tolist(), 0, x, 128, pr.n_pages) for x in range(896)]).T
        pr.q[:, :, 0] = 1.0
        pr.k[page, place, 0, 0] = P.rounded(np.arange(896) * dev, "BF16")
        pr.run()


# One part holds all tiles where the sizes that shape the launch say that there is one: then a tile meets the maximum of those before it
def one_part(n):
    return dict(max_len=1000, max_shared=128, max_group=n)


@pytest.mark.parametrize("n,each", [(8, 4), (16, 4), (30, 4), (60, 4)])
@pytest.mark.parametrize("dev", [0.02, 0.3, 4.0])
def test_scores_that_grow_along_the_positions_of_one_part(p, n, each, dev):
    pr = Problem(p, [n], [900] * n, [896] * n, "BF16", 64, 1, each, 128)
    page, place = np.array([P.cell(pr.tables.tolist(), 0, x, 128, pr.n_pages) for x in range(896)]).T
    pr.q[:, :, 0] = 1.0
    pr.k[page, place, 0, 0] = P.rounded(np.arange(896) * dev, "BF16")
    pr.run(one_part(n))


@pytest.mark.parametrize("n", [7, 14, 30, 60])
@pytest.mark.parametrize("ty,value", [("BF16", 9.0), ("BF16", 89.0), ("F16", 95.0), ("BF16", 200.0), ("F16", 300.0), ("BF16", 3000.0)])
def test_one_position_far_above_the_tiles_before(p, n, ty, value):
    for at in list(range(512, 528)) + [639, 895]:
        pr = Problem(p, [n], [900] * n, [896] * n, ty, 64, 1, 4, 128, scale=1.0)
        page, place = P.cell(pr.tables.tolist(), 0, at, 128, pr.n_pages)
        pr.q[:] = 0.0
        pr.q[:, :, 0] = 1.0
        pr.k[..., 0] *= 0.125
        pr.k[page, place, 0, 0] = value
        pr.run(one_part(n))


@pytest.mark.parametrize("n", [7, 14, 30, 60])
@pytest.mark.parametrize("value", [np.nan, np.inf])
def test_one_score_that_is_no_number(p, n, value):
    for at in list(range(512, 528)) + [3, 895]:
        pr = Problem(p, [n], [900] * n, [896] * n, "BF16", 64, 1, 4, 128)
        page, place = P.cell(pr.tables.tolist(), 0, at, 128, pr.n_pages)
        pr.q[:, :, 0] = 1.0
        pr.k[page, place, 0, 0] = value
        pr.call(one_part(n))(None)
        assert np.isnan(pr.result()).all(), at
        assert b200.load().kernel_error() == 0


def test_a_few_positions_outweigh_all_others(p):
    for at in (0, 127, 128, 500, 767):
        pr = Problem(p, [9], [800] * 9, [768] * 9, "F16", 128, 2, 4, 64)
        page, place = P.cell(pr.tables.tolist(), 0, at, 64, pr.n_pages)
        pr.k[page, place] = P.rounded(pr.k[page, place] * 12, "F16")
        pr.run()


@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("n", [2, 14, 30, 70])
def test_infinities_that_all_rows_see(p, value, n):
    pr = Problem(p, [n], [300 + i for i in range(n)], [256] * n, "BF16", 64, 1, 4, 16)
    page, place = P.cell(pr.tables.tolist(), 0, 77, 16, pr.n_pages)
    pr.v[page, place, 0, 9] = value
    pr.run()


def test_more_groups_than_the_gpu_has_multiprocessors(p):
    n = 340
    Problem(p, [2] * 170, [150 + i % 40 for i in range(n)], [140] * n, "F16", 64, 1, 2, 16).run()


def test_many_heads_a_key_head(p):
    Problem(p, [3], [400, 390, 380], [384] * 3, "BF16", 64, 2, 100, 64, sinks=True).run()


def test_bad_pages_of_the_shared_part_in_every_form(p):
    for n in (4, 12, 28, 70):
        pr = Problem(p, [n], [420 + i % 7 for i in range(n)], [400] * n, "BF16", 128, 1, 4, 32)
        pr.tables[0, 5] = pr.n_pages
        pr.run(error=7)


@pytest.mark.parametrize("n", [5, 14, 30, 70])
def test_a_wait_that_runs_out(p, n):
    """the first CTA of the shared part never asks for its first values: its rows stay as they were, the others' results are those of an undisturbed call"""
    m = b200.load()
    pr = Problem(p, [n, 3], [700 + i for i in range(n + 3)], [640] * (n + 3), "BF16", 128, 2, 4, 64)
    call = pr.call()
    call(None)
    good = pr.result()
    assert m.kernel_error() == 0
    pr.out.upload(P.bits(np.full(pr.q.size + GUARD, -7.0), "BF16"))
    m.lib.b200_debug_attn_wait(20000, 0)
    try:
        call(None)
        m.synchronize()
    finally:
        m.lib.b200_debug_attn_wait(0, -1)
    assert m.kernel_error() == 4 and m.kernel_error() == 0
    got = pr.result()
    rows = min(n, 64)   # of the first block: at most 256 rows of 4 query heads
    assert (got[:rows, :4] == -7.0).all()
    got[:rows, :4] = good[:rows, :4]
    assert np.array_equal(got, good)
    call(None)
    assert np.array_equal(pr.result(), good) and m.kernel_error() == 0


def test_own_positions_are_long(p):
    Problem(p, [2, 2], [2000, 1500, 90, 2222], [40] * 4, "BF16", 128, 2, 4, 16).run()


@pytest.mark.parametrize("hints", [{}, dict(max_len=16, max_shared=16, max_group=1), dict(max_len=100000, max_shared=90000, max_group=200)])
def test_sizes_that_shape_the_launch_are_hints(p, hints):
    Problem(p, [9, 40], [700 + 3 * i for i in range(49)], [650] * 49, "F16", 128, 2, 4).run(hints)
    Problem(p, [], [700, 1, 333], [0] * 3, "F16", 128, 2, 4).run(hints)


def test_sizes_that_shape_the_launch_may_be_the_largest(p):
    Problem(p, [5, 2], [300, 280, 257, 256, 600, 40, 33], [256, 256, 256, 256, 256, 32, 32], "BF16", 64, 2, 2, 16).run(dict(max_len=2 ** 31 - 1, max_shared=2 ** 31 - 1, max_group=2 ** 31 - 1))


def test_wide_scores_and_a_negative_scale(p):
    Problem(p, [6], [500] * 6, [450] * 6, "F16", 128, dev=4.0).run()
    Problem(p, [6], [500] * 6, [450] * 6, "F16", 64, scale=-0.3).run()
    Problem(p, [6], [500] * 6, [450] * 6, "BF16", 64, scale=0.0).run()


def poison(pr, value):
    """every cell that nobody sees"""
    seen = np.zeros((pr.n_pages, pr.page), dtype=bool)
    for g in range(len(pr.first) - 1):
        for s in range(pr.first[g], pr.first[g + 1]):
            for x in range(pr.lens[s]):
                seen[P.cell(pr.tables.tolist(), pr.first[g] if x < pr.shared[s] else s, x, pr.page, pr.n_pages)] = True
    pr.k[~seen] = value
    pr.v[~seen] = value


@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("n", [4, 60])
def test_what_nobody_sees_may_hold_anything(p, value, n):
    pr = Problem(p, [n], [200 + i for i in range(n)], [190] * n, "BF16", 128, 1, 4, 64)
    poison(pr, value)
    pr.run()
    assert np.isfinite(pr.result()).all()


@pytest.mark.parametrize("value", [np.nan, np.inf])
@pytest.mark.parametrize("n", [5, 50])
def test_what_one_row_sees_reaches_no_other(p, value, n):
    # position 150 of the shared part: seen by the rows that are long enough only
    pr = Problem(p, [n], [300 if i % 3 == 0 else 120 for i in range(n)], [256] * n, "F16", 64, 2, 2, 32)
    page, place = P.cell(pr.tables.tolist(), 0, 150, 32, pr.n_pages)
    pr.v[page, place, 1, 5] = value
    pr.run()
    got = pr.result()
    assert np.isfinite(got[1]).all() and not np.isfinite(got[0, 2, 5]) and np.isfinite(got[0, :2]).all()


def test_nan_queries_and_keys_stay_in_their_rows(p):
    pr = Problem(p, [6], [300] * 6, [256] * 6, "BF16", 128, 2, 2)
    pr.q[2, 1, 7] = np.nan
    page, place = P.cell(pr.tables.tolist(), 4, 290, 16, pr.n_pages)
    pr.k[page, place, 1, 0] = np.nan
    pr.run()
    bad = np.isnan(pr.result()).any(2)
    assert bad[2, 1] and bad[4, 2:].all() and bad.sum() == 3


def test_a_row_of_scores_minus_infinity_gives_zeros(p):
    pr = Problem(p, [2], [20, 18], [16] * 2, "BF16", 64, 1, 1)
    pr.q[:] = 0
    pr.q[0, 0, 0] = 1
    pr.k[..., 0] = -np.inf
    pr.k[..., 1:] = 0
    pr.call()(None)
    got = pr.result()
    assert not got[0].any() and np.isnan(got[1]).all()   # 0 * -inf is NaN: that row saw it


def test_pages_out_of_range_are_left_out_and_reported(p):
    for bad, at in ((-1, 2), (10 ** 6, 7), (2 ** 31 - 1, 9)):
        pr = Problem(p, [3], [170, 160, 150], [120] * 3, "F16", 64)
        pr.tables[0, 2 if at == 2 else 1] = bad
        pr.tables[1, min(at, 9)] = bad
        pr.run(error=7)


def test_lengths_beyond_the_table_are_cut_and_reported(p):
    pr = Problem(p, [3], [64, 60, 50], [40] * 3, "F16", 64, table_pages=4)
    pr.lens = [64, 1000, 2 ** 31 - 1]
    pr.call()(None)
    got, pr.lens = pr.result(), [64, 64, 64]
    pr.check(got, 7)


def test_groups_that_do_not_fit_are_reported(p):
    for first in ([0, 9], [1, 4], [0, 3], [0, -2]):
        pr = Problem(p, [4], [64] * 4, [40] * 4, "F16", 64)
        pr.first = first
        pr.call(hints=dict(max_len=64, max_shared=40, max_group=4))(None)
        b200.load().synchronize()
        assert b200.load().kernel_error() == 7


def test_strided_rows(p):
    pr = Problem(p, [3], [64, 60, 50], [40] * 3, "BF16", 64, 2, 3)
    pr.call()
    gap = np.zeros((3, 6, 96))
    gap[:, :, :64] = pr.q
    q, out = device(P.bits(gap, "BF16")), device(P.bits(np.full((6, 3, 72), -7.0), "BF16"))
    call = pr.call()
    call.args.q, call.args.q_nb1, call.args.q_nb2 = q.ptr, 6 * 96 * 2, 96 * 2
    call.args.dst, call.args.dst_nb1, call.args.dst_nb2 = out.ptr, 72 * 2, 3 * 72 * 2   # heads outermost
    call(None)
    got = P.values(out.download(np.uint16, 6 * 3 * 72), "BF16").reshape(6, 3, 72)
    assert (got[:, :, 64:] == -7.0).all()
    pr.check(np.ascontiguousarray(got[:, :, :64].transpose(1, 0, 2)))


def test_pages_that_keys_and_values_share(p):
    # keys and values of a page behind one another, page_stride of both
    pr = Problem(p, [3], [64, 60, 50], [40] * 3, "BF16", 64, 2, 3)
    both = np.concatenate([pr.k.reshape(pr.n_pages, -1), pr.v.reshape(pr.n_pages, -1)], 1)
    store = device(P.bits(both, "BF16"))
    call = pr.call()
    half = 16 * 2 * 64 * 2
    call.args.cache.k, call.args.cache.v, call.args.cache.page_stride = store.ptr, store.ptr + half, 2 * half
    call(None)
    pr.check(pr.result())


def test_the_same_call_gives_the_same_bits(p):
    pr = Problem(p, [20, 3], [900 + i for i in range(23)], [800] * 23, "BF16", 128, 2, 4)
    call = pr.call()
    call(None)
    first = pr.result()
    for _ in range(3):
        call(None)
        assert np.array_equal(first, pr.result())


def test_offsets_beyond_32_bits(p):
    """a pool of over 4 GB: pages behind the 2^32nd byte"""
    m = b200.load()
    page, kv, d = 256, 8, 128
    page_bytes = page * kv * d * 2
    n_pages = (1 << 32) // page_bytes + 6
    rng = np.random.default_rng(0)
    rows = [P.rounded(rng.standard_normal((4, page, kv, d)), "F16") for _ in range(2)]
    store = [m.DeviceBuffer(n_pages * page_bytes) for _ in range(2)]
    for s, a in zip(store, rows):
        s.upload(P.bits(a, "F16"), offset=(n_pages - 4) * page_bytes)
    q = P.rounded(rng.standard_normal((2, 8, d)), "F16")
    tables = np.array([[n_pages - 2, n_pages - 1], [n_pages - 4, n_pages - 3]], dtype=np.int32)
    keep = [device(tables), device(P.bits(q, "F16")), device(np.zeros(q.size, dtype=np.uint16)), device(np.array([300, 400], dtype=np.int32)), device(np.array([256, 256], dtype=np.int32)), device(np.array([0, 2], dtype=np.int32))]
    cache = p.Cache(p.F16, page, n_pages, kv, d, store[0].ptr, store[1].ptr, keep[0].ptr, 2, 2)
    p.PrefixAttn(cache, 2, 8, keep[1].ptr, keep[2].ptr, keep[3].ptr, d ** -0.5, shared=keep[4].ptr, group_first=keep[5].ptr, n_group=1, max_len=400, max_shared=256, max_group=2)(None)
    got = P.values(keep[2].download(np.uint16, q.size), "F16").reshape(q.shape)
    want, size, _, _ = P.attention(rows[0], rows[1], (tables - (n_pages - 4)).tolist(), q, [300, 400], [256, 256], [0, 2], d ** -0.5)
    assert (np.abs(got - want) <= (2 * P.HALF_STEP["F16"] + 1e-3) * size).all() and m.kernel_error() == 0
