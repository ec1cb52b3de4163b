"""b200_beam_select over the whole range of its logits and scores, against the definition in 64 bits; the bounds are those of test_gpu_beam.py: a subtraction of a chunk's
maximum is exact where it counts (words within a factor of two of it, or within 2^-24 of a distance that a weight of exp(-distance) feels)."""
import numpy as np
import pytest

import b200
import plain_paged as P
from test_gpu_beam import head, p, select  # noqa: F401

pytestmark = pytest.mark.gpu

# requests, beams, vocabulary: one launch of clusters, two launches
FORMS = [(2, 3, 5000), (2, 9, 20000)]
FAR = [4095.0, 4097.0, 1e4, 65504.0, 1e6, 1e8, 1e9, 1e10, 1e12, 1e20, 1e29, 2e30, 3e38]


@pytest.mark.parametrize("R,B,V", FORMS)
@pytest.mark.parametrize("ty", ["F32", "BF16"])
@pytest.mark.parametrize("mask", [-x for x in FAR])
def test_words_masked_with_a_finite_value(p, R, B, V, ty, mask):
    rng = np.random.default_rng(int(-mask) % 1000)
    x = head(rng, R, B, V, ty)
    spread = np.full_like(x, P.rounded(mask, ty))
    spread[..., 5::V // 11] = x[..., 5::V // 11]      # a dozen words are allowed
    select(p, spread, -rng.random((R, B)), 8, ty)
    side = np.full_like(x, P.rounded(mask, ty))
    side[..., 40:52] = x[..., 40:52]                  # all in a row's first chunk: the others are masked as a whole
    select(p, side, -rng.random((R, B)), 8, ty)
    select(p, side[:1, :1], -rng.random((1, 1)), 20, ty)   # fewer than are asked for: masked ones follow


@pytest.mark.parametrize("R,B,V", FORMS)
@pytest.mark.parametrize("ty", ["F32", "BF16"])
@pytest.mark.parametrize("value", FAR)
def test_one_word_far_above_the_others(p, R, B, V, ty, value):
    rng = np.random.default_rng(int(value) % 1000)
    x = head(rng, R, B, V, ty)
    x[..., V // 3] = P.rounded(value, ty)
    select(p, x, -rng.random((R, B)), B, ty)
    if value <= 1e9:   # further away 64 bits do not tell the others' scores apart
        select(p, x, -rng.random((R, B)), B + 8, ty)


@pytest.mark.parametrize("R,B,V", FORMS)
@pytest.mark.parametrize("sign", [-1.0, 1.0])
@pytest.mark.parametrize("ty,value", [("F16", 30000.0), ("F16", 65504.0)] + [(ty, x) for ty in ("F32", "BF16") for x in FAR])
def test_rows_of_one_value_and_around_it(p, R, B, V, ty, sign, value):
    rng = np.random.default_rng(int(value) % 1000)
    flat = np.full((R, B, V), P.rounded(sign * value, ty))
    select(p, flat, -rng.random((R, B)), 8, ty)
    if value <= 1e9:
        most = np.finfo(np.float16).max if ty == "F16" else np.inf
        select(p, P.rounded(np.clip(flat + head(rng, R, B, V), -most, most), ty), -rng.random((R, B)), 8, ty)


def test_the_sum_is_as_good_far_from_zero(p):
    # words at distances of 0 to 8 from offsets on both sides of where a chunk's exponentials change their form
    rng = np.random.default_rng(3)
    for offset in (-65000.0, -4200.0, -4096.0, -4090.0, 4088.0, 4096.0, 4104.0, 60000.0):
        for R, B, V in FORMS:
            x = P.rounded(offset - 8.0 * rng.random((R, B, V)), "F32")
            select(p, x, -rng.random((R, B)), 4)


def chosen(p, x, scores, k):
    """F32 logits [requests, beams, vocab] -> (scores, tokens, parents), held to the definition; scores may be infinite"""
    m = b200.load()
    R, B, V = x.shape
    scores = np.asarray(scores, dtype=np.float32)
    keep = [m.device_array(np.ascontiguousarray(x, dtype=np.float32)), m.device_array(scores)]
    outs = [m.device_array(np.full(R * k, 77, dtype=np.int32)) for _ in range(3)]
    p.BeamSelect(p.F32, R, B, V, k, keep[0].ptr, keep[1].ptr, *(o.ptr for o in outs))(None)
    s, w, b = (o.download(np.int32, R * k).reshape(R, k) for o in outs)
    s = s.view(np.float32).astype(np.float64)
    for r in range(R):
        found = []
        for j in range(B):
            v = x[r, j].astype(np.float32).astype(np.float64)
            if not scores[r, j] > -np.inf or v.max() == -np.inf:
                continue
            with np.errstate(invalid="ignore"):
                off = np.where(v == v.max(), 0.0, v - v.max())
                gain = float(scores[r, j]) + (off - np.log(np.exp(off).sum()))
            best = np.lexsort((np.arange(V), -v, -gain))[:k]   # NaN (none of the words beside one of +inf) comes last
            found += [(-gain[t], j, -v[t], int(t)) for t in best if gain[t] > -np.inf]
        found = sorted(found)[:k]
        n = len(found)
        assert [(f[1], f[3]) for f in found] == list(zip(b[r, :n].tolist(), w[r, :n].tolist()))
        want = -np.array([f[0] for f in found])
        assert ((np.abs(s[r, :n] - want) <= 2.0 ** -23 * np.abs(want) + 2.0 ** -20) | (s[r, :n] == want)).all()
        assert (s[r, n:] == -np.inf).all() and (w[r, n:] == -1).all() and (b[r, n:] == -1).all()
    assert m.kernel_error() == 0
    return s, w, b


@pytest.mark.parametrize("R,B,V", FORMS)
def test_beams_of_infinite_scores(p, R, B, V):
    # a score of +inf keeps its beam's words in front; beside a logit of +inf no other word is a candidate, whatever the score
    rng = np.random.default_rng(21)
    x = head(rng, R, B, V)
    x[:, 0, ::V // 5] = np.inf
    x[:, 1] = -np.inf
    x[:, 1, 77:80] = 1.0
    scores = -rng.random((R, B))
    scores[0, :2] = np.inf
    chosen(p, x, scores, 12)
    chosen(p, x[:, :2], scores[:, :2], 40)


@pytest.mark.parametrize("R,B,V", FORMS + [(1, 1, 30000), (3, 20, 9000)])
@pytest.mark.parametrize("score", [-1e9, -1e16, -1e20, -3e38, 1e18, 1e20, 3e38, np.inf])
def test_scores_beside_which_logits_are_small(p, R, B, V, score):
    # beams that a program has put far behind (or before) the others: 64 bits do not tell their words' scores apart, their logits do
    rng = np.random.default_rng(22)
    x = head(rng, R, B, V)
    # beams one behind the other, where 64 bits keep some of what a logit adds; else all alike
    scores = np.full((R, B), score) * (1.0 + np.arange(B) if abs(score) <= 1e18 else 1.0)
    chosen(p, x, scores, 12)
    scores[:, 0] = -2.0
    x[:, 0] = -np.inf
    x[:, 0, 17:20] = 3.0        # the beam in front has three words
    chosen(p, x, scores, 40)
    chosen(p, P.rounded(rng.integers(0, 3, x.shape).astype(np.float64), "F32"), scores, 30)


@pytest.mark.parametrize("R,B,V", FORMS)
@pytest.mark.parametrize("size", [1e-18, 1e-30, 1e-44])
def test_logits_too_small_to_change_a_score(p, R, B, V, size):
    rng = np.random.default_rng(23)
    x = P.rounded(rng.standard_normal((R, B, V)) * size, "F32")
    chosen(p, x, np.full((R, B), -1.0), 9)
    x[:, :, 11] = 5.0
    chosen(p, x, -rng.random((R, B)), 50)
    chosen(p, x, np.full((R, B), -1.0), 50)


def test_ended_beams_among_equal_scores(p):
    m = b200.load()
    x = np.zeros((1, 3, 4000), dtype=np.float32)
    x[0, 2, 3999] = 100.0                     # as good as certain: 64 bits give the score of the ended beam
    outs = [m.device_array(np.full(4, 77, dtype=np.int32)) for _ in range(3)]
    keep = [m.device_array(x), m.device_array(np.array([-3.0, -2.0, -2.0], dtype=np.float32)), m.device_array(np.array([0, 1, 0], dtype=np.uint8))]
    p.BeamSelect(p.F32, 1, 3, 4000, 4, keep[0].ptr, keep[1].ptr, *(o.ptr for o in outs), done=keep[2].ptr, end_token=3000)(None)
    assert outs[1].download(np.int32, 4).tolist() == [3000, 3999, 0, 1] and outs[2].download(np.int32, 4).tolist() == [1, 2, 0, 0]


@pytest.mark.parametrize("R,B,V", [(147, 1, 2100), (148, 1, 2100), (149, 1, 2100), (298, 1, 900), (13, 4, 8000), (14, 4, 8000), (15, 4, 8000), (16, 4, 8000), (64, 8, 700)])
def test_as_many_requests_as_either_form_takes(p, R, B, V):
    rng = np.random.default_rng(R)
    select(p, head(rng, R, B, V), -rng.random((R, B)), 2 * B)
    select(p, head(rng, R, B, V, "BF16"), -rng.random((R, B)), B, "BF16", done=(rng.random((R, B)) < 0.2).astype(int), end=5)
