"""b200_beam_select and b200_beam_reorder against their definitions.  Scores: F32 sums of exponentials each good to 2^-21 (so the logarithm is), one rounding of the
score; tokens and parents are equal, ties included."""
import importlib

import numpy as np
import pytest

import b200
import plain_paged as P

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def p():
    b200.load()
    return importlib.import_module("llama_rust_b200.paged")


def device(a):
    return b200.load().device_array(a)


def select(p, logits, scores, k, ty="F32", done=None, end=0, pad=0, off=0):
    """logits: values of the type [requests, beams, vocab]; pad: elements between rows; off: elements before the first"""
    R, B, V = logits.shape
    scores = np.asarray(scores, dtype=np.float32)
    TY = {"F32": p.F32, "F16": p.F16, "BF16": p.BF16}
    flat = np.full((R * B, V + pad), 1e4)
    flat[:, :V] = logits.reshape(R * B, V)
    size = 4 if ty == "F32" else 2
    x = device(P.bits(np.concatenate([np.full(off, 1e4), flat.reshape(-1)])[: off + R * B * (V + pad) - pad], ty))
    keep = [device(scores), device(np.zeros((R, B), dtype=np.uint8) if done is None else np.asarray(done, dtype=np.uint8))]
    outs = [device(np.full(R * k + 16, 77, dtype=np.int32)) for _ in range(3)]
    p.BeamSelect(TY[ty], R, B, V, k, x.ptr + off * size, keep[0].ptr, outs[0].ptr, outs[1].ptr, outs[2].ptr, done=None if done is None else keep[1].ptr, end_token=end, logits_ld=V + pad)(None)
    got = [o.download(np.int32, R * k + 16) for o in outs]
    for g in got:
        assert (g[R * k:] == 77).all()
    s, w, b = got[0][: R * k].view(np.float32).reshape(R, k).astype(np.float64), got[1][: R * k].reshape(R, k), got[2][: R * k].reshape(R, k)
    want = P.select(logits, scores.astype(np.float64), k, done, end)
    assert np.array_equal(w, want[1]) and np.array_equal(b, want[2])
    live = want[0] > -np.inf
    assert (s[~live] == -np.inf).all()
    assert (np.abs(s - want[0])[live] <= 2.0 ** -23 * np.abs(want[0])[live] + 2.0 ** -20).all()
    assert b200.load().kernel_error() == 0
    return s, w, b


def head(rng, R, B, V, ty="F32"):
    x = rng.standard_normal((R, B, V)) * 2
    x[..., ::61] *= 2.5
    return P.rounded(x, ty)


@pytest.mark.parametrize("ty", ["F32", "F16", "BF16"])
@pytest.mark.parametrize("V", [1, 2, 31, 1000, 2047, 2048, 2049, 8193, 50001])
def test_vocabularies(p, ty, V):
    rng = np.random.default_rng(V)
    select(p, head(rng, 3, 4, V, ty), -5 * rng.random((3, 4)), 8, ty)


@pytest.mark.parametrize("B,k", [(1, 1), (1, 5), (2, 4), (7, 7), (16, 32), (33, 64), (64, 64), (64, 128), (5, 128)])
def test_beams_and_candidates(p, B, k):
    rng = np.random.default_rng(B * 1000 + k)
    select(p, head(rng, 2, B, 3001), -5 * rng.random((2, B)), k)


def test_many_rows_take_long_chunks(p):
    rng = np.random.default_rng(9)
    select(p, head(rng, 40, 4, 20011), -5 * rng.random((40, 4)), 8)
    select(p, head(rng, 40, 4, 20011, "BF16"), -5 * rng.random((40, 4)), 8, "BF16")


def test_a_large_vocabulary(p):
    rng = np.random.default_rng(12)
    select(p, head(rng, 1, 2, 1000003), -rng.random((1, 2)), 128)
    select(p, head(rng, 1, 2, 1000003, "F16"), -rng.random((1, 2)), 4, "F16")


@pytest.mark.parametrize("k", [15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128])
@pytest.mark.parametrize("B,V", [(2, 9001), (9, 20000)])
def test_where_the_best_logits_lie(p, k, B, V):
    # spread out; side by side, so that one thread's and one group's values are the best; few that are finite
    rng = np.random.default_rng(k)
    x = head(rng, 2, B, V)
    select(p, x, -rng.random((2, B)), k)
    side = np.sort(x, axis=-1)
    select(p, side, -rng.random((2, B)), k)
    few = np.full_like(x, -np.inf)
    few[..., ::V // 20] = x[..., ::V // 20]
    select(p, few, -rng.random((2, B)), k)


@pytest.mark.parametrize("offset", [0.0, 30.0, -500.0, 2000.0])
def test_logits_far_from_zero(p, offset):
    # x log2(e) is rounded once for a chunk's maximum: what that is off by must not show
    rng = np.random.default_rng(13)
    x = P.rounded(head(rng, 2, 3, 20000) + offset, "F32")
    select(p, x, -rng.random((2, 3)), 8)


def test_one_word_has_nearly_all_the_probability(p):
    rng = np.random.default_rng(14)
    x = head(rng, 2, 3, 9000)
    x[:, :, 4321] = 60.0
    select(p, P.rounded(x, "F32"), -rng.random((2, 3)), 6)


@pytest.mark.parametrize("ty,V,pad,off", [("F32", 999, 1, 0), ("F32", 999, 0, 1), ("F32", 1024, 2, 3), ("BF16", 999, 1, 1), ("BF16", 1003, 0, 7), ("F16", 4096, 5, 3), ("BF16", 4095, 0, 0)])
def test_rows_at_any_address(p, ty, V, pad, off):
    rng = np.random.default_rng(V)
    select(p, head(rng, 2, 5, V, ty), -rng.random((2, 5)), 6, ty, pad=pad, off=off)


def test_the_same_rows_give_the_same_scores_wherever_they_lie(p):
    rng = np.random.default_rng(1)
    for ty, V in (("F32", 5003), ("BF16", 40001)):
        one = head(rng, 1, 1, V, ty)
        s, w, b = select(p, np.repeat(one, 4, 1), np.full((1, 4), -1.0), 12, ty)   # equal beams: their first tokens in the order of the beams
        assert list(b[0, :4]) == [0, 1, 2, 3] and len(set(w[0, :4])) == 1 and len(set(s[0, :4])) == 1


@pytest.mark.parametrize("ty", ["F32", "F16"])
@pytest.mark.parametrize("V,k", [(3000, 8), (40000, 128), (100, 128)])
def test_equal_logits_go_by_token(p, ty, V, k):
    select(p, np.zeros((1, 2, V)), np.array([[-1.0, -1.0]]), k, ty)
    x = np.zeros((1, 2, V))
    x[0, 0, V // 2:] = 1.0
    x[0, 1, 7::3] = 1.0
    select(p, x, np.array([[-1.0, -1.0]]), k, ty)
    x[0, :, 5] = 3.0
    x[0, :, 6] = -0.0
    select(p, x, np.array([[-1.0, -2.0]]), k, ty)


def test_few_values_many_times(p):
    rng = np.random.default_rng(2)
    for V in (9000, 33000):
        select(p, rng.integers(0, 3, (2, 3, V)).astype(np.float64), -rng.random((2, 3)), 20)


def test_masked_words(p):
    rng = np.random.default_rng(5)
    x = head(rng, 2, 3, 5000)
    x[rng.random(x.shape) < 0.999] = -np.inf      # a few words are allowed
    x[0, 1] = -np.inf                             # none of a beam's
    x[1, 2, 4000:] = np.nan
    select(p, x, -rng.random((2, 3)), 16)
    x[:] = -np.inf
    s, w, b = select(p, x, -rng.random((2, 3)), 3)
    assert (w == -1).all() and (b == -1).all()
    x[1, 1, 17] = 2.0                             # the only candidate there is
    select(p, x, -rng.random((2, 3)), 3)


def test_infinite_and_lowest_logits(p):
    rng = np.random.default_rng(6)
    x = head(rng, 1, 3, 3000)
    x[0, 0, [5, 900]] = np.inf
    x[0, 1] = np.finfo(np.float32).min
    x[0, 1, 3] = 0.0
    x[0, 2] = np.finfo(np.float32).min            # all the lowest value: even probabilities
    select(p, x, np.array([[-3.0, -1.0, -2.0]]), 10)


def test_beams_without_a_score(p):
    rng = np.random.default_rng(7)
    x = head(rng, 2, 4, 3000)
    s, w, b = select(p, x, np.array([[0.0, -np.inf, -np.inf, -np.inf], [np.nan, -1.0, np.nan, -2.0]]), 8)   # the first step of a search
    assert (b[0] == 0).all() and set(b[1]) <= {1, 3}


def test_beams_that_have_ended(p):
    rng = np.random.default_rng(8)
    x = head(rng, 3, 4, 3000)
    x[0, 0] = np.nan                              # nothing of an ended beam's row is read
    done = np.array([[1, 0, 0, 0], [0, 2, 0, 1], [1, 1, 1, 1]])
    s, w, b = select(p, x, -3 * rng.random((3, 4)), 6, done=done, end=17)
    assert (w[2, :4] == 17).all() and (w[2, 4:] == -1).all()


def test_scores_far_apart(p):
    rng = np.random.default_rng(10)
    select(p, head(rng, 2, 4, 3000), np.array([[-1.0, -500.0, -30.0, -2.0], [-1e6, -2e6, -1e6 - 1, -1.5e6]]), 16)


# ---- reorder ---------------------------------------------------------------------------------------------------------------------------------

def reorder(p, parents, lens, shared_pages=2, pages=5, page_size=16, n_pools=3, page_bytes=1024, gap=0, seed=0, row_of=True, bad=None):
    m = b200.load()
    rng = np.random.default_rng(seed)
    R, B = np.asarray(parents).shape
    n = R * B
    n_pages = R * shared_pages + n * (pages - shared_pages) + 1
    ids = rng.permutation(n_pages)
    tables = np.concatenate([ids[: R * shared_pages].reshape(R, 1, shared_pages).repeat(B, 1).reshape(n, shared_pages),
                             ids[R * shared_pages: n_pages - 1].reshape(n, pages - shared_pages)], 1).astype(np.int32)
    if bad:
        tables[bad[0], bad[1]] = bad[2]
    stride = page_bytes + gap
    pools = [rng.integers(0, 256, (n_pages, stride), dtype=np.uint8) for _ in range(n_pools)]
    want = P.reorder(np.asarray(parents).tolist(), tables.tolist(), list(lens), page_size, [x[:, :page_bytes] for x in pools])
    dp = [device(x) for x in pools]
    keep = [device(np.asarray(parents, dtype=np.int32)), device(tables), device(np.asarray(lens, dtype=np.int32))]
    outs = [device(np.full(x + 8, 77, dtype=np.int32)) for x in (n * pages, n, n)]
    p.BeamReorder(R, B, keep[0].ptr, keep[1].ptr, outs[0].ptr, pages, keep[2].ptr, outs[1].ptr, outs[2].ptr if row_of else None, page_size, n_pages, page_bytes, [d.ptr for d in dp],
                  page_stride=stride if gap else 0)(None)
    got = [o.download(np.int32, c + 8) for o, c in zip(outs, (n * pages, n, n))]
    for g, c in zip(got, (n * pages, n, n)):
        assert (g[c:] == 77).all()
    assert np.array_equal(got[0][: n * pages].reshape(n, pages), np.array(want[0])) and np.array_equal(got[1][:n], want[1])
    if row_of:
        assert np.array_equal(got[2][:n], want[2])
    else:
        assert (got[2] == 77).all()
    for d, before, after in zip(dp, pools, want[3]):
        x = d.download(np.uint8, n_pages * stride).reshape(n_pages, stride)
        assert np.array_equal(x[:, :page_bytes], after) and np.array_equal(x[:, page_bytes:], before[:, page_bytes:])
    return m.kernel_error()


@pytest.mark.parametrize("B", [1, 2, 3, 8, 32, 33, 64])
@pytest.mark.parametrize("spread", [1, 3, 64])
def test_any_parents(p, B, spread):
    rng = np.random.default_rng(B + spread)
    R = 3
    parents = np.minimum(rng.integers(0, spread, (R, B)), B - 1)
    assert reorder(p, parents, rng.integers(0, 81, R * B)) == 0


def test_beams_not_in_use(p):
    assert reorder(p, [[2, -1, 2, -5], [-1, -1, -1, -1], [0, 1, 2, 3], [3, 2, 1, 0], [-1, 0, 0, 0]], [80] * 20) == 0


@pytest.mark.parametrize("lens", [0, 1, 31, 32, 33, 48, 49, 80])
def test_only_pages_in_use_move(p, lens):
    assert reorder(p, [[0, 0, 1, 1], [3, 3, 3, 3]], [lens] * 8) == 0


@pytest.mark.parametrize("page_bytes,gap", [(16, 0), (48, 16), (4096 + 16, 0), (32768, 0), (32768 + 16, 0), (3 * 32768, 64), (262144, 0)])
def test_page_sizes(p, page_bytes, gap):
    assert reorder(p, [[1, 1, 0], [2, 2, 2]], [70] * 6, page_bytes=page_bytes, gap=gap) == 0


@pytest.mark.parametrize("n_pools", [0, 1, 128, 129, 300])
def test_numbers_of_pools(p, n_pools):
    assert reorder(p, [[1, 1, 0, 0]], [70] * 4, n_pools=n_pools, page_bytes=64) == 0


def test_recurrent_states_are_pages(p):
    assert reorder(p, [[1, 1, 3, 3], [0, 0, 0, 0]], [1] * 8, shared_pages=0, pages=1, page_size=1, page_bytes=4 * 20 * 12) == 0


def test_row_of_may_be_left_out(p):
    assert reorder(p, [[1, 1, 0]], [70] * 3, row_of=False) == 0


def test_indices_out_of_range_are_reported(p):
    assert reorder(p, [[4, 0, 0, 0], [1, 1, 9, 1]], [80] * 8) == 7            # parents: the beam counts as not in use
    assert reorder(p, [[1, 1, 0]], [70, 70, 70], bad=(1, 3, -1)) == 7          # a page of the parent's
    assert reorder(p, [[1, 1, 0]], [70, 70, 70], bad=(2, 4, 10 ** 7)) == 7     # a page of the row that is taken
    assert reorder(p, [[1, 1, 0]], [70, 1000, 70]) == 7                        # more positions than the row has pages
    assert reorder(p, [[1, 1, 0]], [70, -3, 70]) == 0
