"""b200_beam_select over the whole range of its logits and scores, against the definition in 64 bits; the bounds are those of test_gpu_beam.py: a subtraction of a chunk's
maximum is exact where it counts (words within a factor of two of it, or within 2^-24 of a distance that a weight of exp(-distance) feels)."""
import numpy as np
import pytest

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
