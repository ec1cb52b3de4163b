"""b200_prefix_attn where scores are so large that F32 holds whole steps of their logarithm only.  One channel of q and k makes the scores, all of them exact in F32 and far
apart, so that the best position has all the weight and the result is its value (of two equal best ones the mean).  The bound: its weight may be rounded to the cache's type, half a
step of it, the result is rounded once more, and F32 sums and quotients are good to 2^-20:  |got - o| <= (half + 2^-20) mean |v| + half |o| + SMALLEST."""
import numpy as np
import pytest

import b200
import plain_paged as P
from test_gpu_prefix_attn import Problem, one_part, p  # noqa: F401

pytestmark = pytest.mark.gpu


made = {}   # problems by what shapes them: their values take longer to make than a call


def outstanding(p, n, ty, d, factor, value, scale, ats, hints, page=64):
    """queries with `factor` in channel 0, keys with `value` there at positions `ats`, further below at the others"""
    if (n, ty, d) not in made:
        made[n, ty, d] = Problem(p, [n], [900] * n, [896] * n, ty, d, 1, 4, page)
    pr = made[n, ty, d]
    pr.p, pr.scale = p, scale
    pr.q[:] = 0.0
    pr.q[..., 0] = factor
    low = 0.5 * value if factor * value * scale > 0 else 2.0 * value
    pr.k[..., 0] = P.rounded(low * (1.0 + (np.arange(pr.k[..., 0].size).reshape(pr.k[..., 0].shape) % 5) * (-0.0625 if low * factor * scale > 0 else 0.0625)), ty)
    assert (pr.k[..., 0] * factor * scale <= value * factor * scale - 0.25 * abs(value * factor * scale)).all()
    cells = []
    for at in ats:
        page_id, place = P.cell(pr.tables.tolist(), 0, at, page, pr.n_pages)
        pr.k[page_id, place, 0, 0] = float(P.rounded(value, ty).item())
        cells.append(pr.v[page_id, place, 0])
    pr.call(hints)(None)
    want, size = sum(cells) / len(cells), sum(map(np.abs, cells)) / len(cells)
    got = pr.result()
    assert b200.load().kernel_error() == 0
    half = P.HALF_STEP[ty]
    assert (np.abs(got - want) <= (half + 2.0 ** -20) * size + half * np.abs(want) + P.SMALLEST[ty]).all(), (ats, got[0, 0, :4], want[:4])


ROWS = [7, 14, 30, 60]   # times four heads: every form of the shared part


@pytest.mark.parametrize("n", ROWS)
@pytest.mark.parametrize("value", [1e6, 1.1e7, 1.2e7, 2.9e8, 3.1e9, 1e10, 7.5e10, 1e15, 1e20, 1e30])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_scores_of_bf16(p, n, value, sign):
    for hints in (True, one_part(n)):
        for ats in ([5], [400, 640], [895]):
            outstanding(p, n, "BF16", 128, 1.0, sign * value, 1.0, ats, hints)


@pytest.mark.parametrize("n", ROWS)
@pytest.mark.parametrize("value", [300.0, 8848.0, 13264.0, 22880.0, 65504.0])
@pytest.mark.parametrize("scale", [1.0, -1.0, 0.125, 512.0])
def test_scores_of_f16(p, n, value, scale):
    for hints in (True, one_part(n)):
        for ats in ([5], [400, 640], [895]):
            for sign in (1.0, -1.0):
                if value <= 32752.0 or sign * scale > 0:
                    outstanding(p, n, "F16", 64, 2.0 ** 15, sign * value, scale, ats, hints)


def test_best_positions_of_a_row_s_own(p):
    # far behind them the shared ones
    for value in (3.1e9, 1e10, 1e20):
        outstanding(p, 9, "BF16", 64, 1.0, value, 1.0, [3], dict(max_len=900, max_shared=100, max_group=9))
        outstanding(p, 9, "BF16", 64, 1.0, -value, 1.0, [3], dict(max_len=900, max_shared=100, max_group=9))


@pytest.mark.parametrize("n", [2, 30])
def test_sinks_at_the_ends_of_their_range(p, n):
    # the largest take all the weight, the lowest none of it
    most = float(np.finfo(np.float32).max)
    pr = Problem(p, [n], [300 + i for i in range(n)], [256] * n, "BF16", 64, 1, 4, 16, sinks=True)
    pr.sinks[:] = [most, 2.5e38, -most, -np.inf]
    pr.run()
    got = pr.result()
    assert not got[:, :2].any() and got[:, 2:].any()


@pytest.mark.parametrize("n", [3, 40])
def test_outputs_in_the_place_of_the_queries(p, n):
    # rows that are computed again read their queries after others have been stored
    pr = Problem(p, [n], [300 + i for i in range(n)], [256] * n, "BF16", 128, 1, 4, 16)
    page, place = P.cell(pr.tables.tolist(), 0, 77, 16, pr.n_pages)
    pr.v[page, place, 0, 9] = np.inf
    pr.q[1, 2, 0] = 2.0 ** 30
    call = pr.call()
    call.args.dst = call.args.q
    call(None)
    pr.out = pr.keep[3]
    got = P.values(pr.out.download(np.uint16, pr.q.size), pr.ty).reshape(pr.q.shape)
    apart = pr.call()
    apart(None)
    assert np.array_equal(got, pr.result(), equal_nan=True) and b200.load().kernel_error() == 0


def long_tail(p, ty, n, shared, length, peaks, steps, hints, page=256, each=4):
    """`length` positions of which those in `peaks` outweigh each of the others by 2^steps, the others' values being 1 where the peaks' are 0: channels 0 .. 31 hold the others' share of the
    weight, channels 32 .. 63 the peaks'.  Pages are named many times over"""
    m = b200.load()
    d, heads = 64, each
    score = float(P.rounded(steps * np.log(2.0), ty).item())
    k, v = np.zeros((2, page, 1, d)), np.zeros((2, page, 1, d))
    k[0, peaks, 0, 0] = score
    v[..., :32] = 1.0
    v[0, peaks, 0, :32], v[0, peaks, 0, 32:] = 0.0, 1.0
    q = np.zeros((n, heads, d))
    q[..., 0] = 1.0
    tables = np.ones((n, length // page), dtype=np.int32)
    tables[:, 0] = 0
    keep = [m.device_array(x) for x in (P.bits(k, ty), P.bits(v, ty), tables, P.bits(q, ty), np.zeros(q.size, dtype=np.uint16), np.full(n, length, dtype=np.int32), np.full(n, shared, dtype=np.int32), np.array([0, n], dtype=np.int32))]
    cache = p.Cache({"F16": p.F16, "BF16": p.BF16}[ty], page, 2, 1, d, keep[0].ptr, keep[1].ptr, keep[2].ptr, length // page, n)
    p.PrefixAttn(cache, n, heads, keep[3].ptr, keep[4].ptr, keep[5].ptr, 1.0, shared=keep[6].ptr, group_first=keep[7].ptr, n_group=1, **hints)(None)
    got = P.values(keep[4].download(np.uint16, q.size), ty).reshape(q.shape)
    rest = (length - len(peaks)) * np.exp(-score)
    want = np.repeat([rest / (len(peaks) + rest), len(peaks) / (len(peaks) + rest)], 32)
    # equal weights: all are rounded alike, by half a step; the result once more; scores and exponentials are good to 2^-20; an output grows in 4096 additions of 16
    # products, each off by at most 2^-23 of what it has come to: 2^-12 of the whole
    half = P.HALF_STEP[ty]
    assert (np.abs(got - want) <= (2 * half + 2.0 ** -19 + 2.0 ** -12) * want + P.SMALLEST[ty]).all(), (got[0, 0, [0, 63]], want[[0, 63]])
    assert m.kernel_error() == 0


@pytest.mark.parametrize("ty", ["F16", "BF16"])
@pytest.mark.parametrize("steps", [10.0, 15.3, 19.7])
@pytest.mark.parametrize("n", ROWS)
def test_many_small_weights_behind_a_shared_position(p, ty, steps, n):
    long_tail(p, ty, n, 65536, 65536, [0, 128], steps, dict(max_len=1000, max_shared=128, max_group=n))


@pytest.mark.parametrize("ty", ["F16", "BF16"])
@pytest.mark.parametrize("steps", [10.0, 15.3, 19.7, 25.4, 27.8])
def test_many_small_weights_behind_a_position_of_a_row_s_own(p, ty, steps):
    long_tail(p, ty, 2, 0, 65536, [0, 16, 32, 48], steps, dict(max_len=64, max_shared=0, max_group=0))


@pytest.mark.parametrize("n", ROWS)
def test_small_weights_of_f16_that_are_rounded_to_whole_steps(p, n):
    # below 2^-22 of the largest a weight is a multiple of 2^-32 of it: that bounds what a tail may lose, 2^-33 a position
    m, length = b200.load(), 65536
    for steps in (23.3, 25.4, 28.6):
        page, d, heads, score = 256, 64, 4, float(P.rounded(steps * np.log(2.0), "F16").item())
        k, v = np.zeros((2, page, 1, d)), np.ones((2, page, 1, d))
        k[0, [0, 128], 0, 0], v[0, [0, 128]] = score, 0.0
        q = np.zeros((n, heads, d))
        q[..., 0] = 1.0
        tables = np.ones((n, length // page), dtype=np.int32)
        tables[:, 0] = 0
        keep = [m.device_array(x) for x in (P.bits(k, "F16"), P.bits(v, "F16"), tables, P.bits(q, "F16"), np.zeros(q.size, dtype=np.uint16), np.full(n, length, dtype=np.int32), np.full(n, length, dtype=np.int32), np.array([0, n], dtype=np.int32))]
        cache = p.Cache(p.F16, page, 2, 1, d, keep[0].ptr, keep[1].ptr, keep[2].ptr, length // page, n)
        p.PrefixAttn(cache, n, heads, keep[3].ptr, keep[4].ptr, keep[5].ptr, 1.0, shared=keep[6].ptr, group_first=keep[7].ptr, n_group=1, max_len=1000, max_shared=128, max_group=n)(None)
        got = P.values(keep[4].download(np.uint16, q.size), "F16")
        rest = (length - 2) * np.exp(-score)
        want = rest / (2.0 + rest)
        assert (np.abs(got - want) <= length * 2.0 ** -33 / 2.0 + 2.0 ** -10 * want + P.SMALLEST["F16"]).all(), (steps, got[0], want)
    assert m.kernel_error() == 0
