"""Outputs of b200_beam_select that lie on other operands: refused before anything touches a device, but for the new scores in the place of as many old ones."""
import importlib

import pytest

import b200

A = 1 << 24   # addresses that nobody reads here, further apart than any operand is long
R, B, V = 2, 4, 1000


@pytest.fixture(scope="module")
def p():
    b200.load()
    return importlib.import_module("llama_rust_b200.paged")


def message(p, **kw):
    a = dict(logits_type=p.F32, n_request=R, n_beam=B, n_vocab=V, k=B, logits=A, scores=2 * A, done=3 * A, out_scores=4 * A, out_tokens=5 * A, out_parents=6 * A, workspace=(7 * A, 1 << 20))
    a.update(kw)
    with pytest.raises(Exception) as e:   # these addresses are refused in any case, further on
        p.BeamSelect(**a)(None)
    return str(e.value)


def test_operands_apart_are_no_overlap(p):
    assert "overlaps" not in message(p)
    # side by side
    assert "overlaps" not in message(p, out_scores=2 * A + 4 * R * B, out_tokens=2 * A + 8 * R * B, out_parents=2 * A - 4 * R * B)
    assert "overlaps" not in message(p, out_tokens=A + 4 * R * B * V, done=None, out_parents=3 * A)


def test_new_scores_may_take_the_place_of_as_many_old_ones(p):
    assert "overlaps" not in message(p, out_scores=2 * A)


@pytest.mark.parametrize("k", [1, 3, 5, 8])
def test_new_scores_in_the_place_of_more_or_fewer_are_refused(p, k):
    assert "overlaps" in message(p, k=k, out_scores=2 * A)


@pytest.mark.parametrize("kw", [
    dict(out_scores=2 * A + 4), dict(out_scores=2 * A - 4), dict(out_tokens=2 * A), dict(out_parents=2 * A + 4 * R * B - 4), dict(out_scores=3 * A), dict(out_tokens=3 * A + 4), dict(out_scores=A), dict(out_parents=A + 4 * (R * B * V - 1)),
    dict(out_tokens=4 * A), dict(out_parents=4 * A + 4), dict(out_parents=5 * A), dict(out_scores=7 * A), dict(out_tokens=7 * A + 256), dict(workspace=(2 * A, 1 << 20)), dict(workspace=(A, 1 << 20)),
    dict(workspace=(3 * A - 256, 1 << 20)), dict(out_scores=2 * A, out_tokens=2 * A)])
def test_other_overlaps_are_refused(p, kw):
    text = message(p, **kw)
    assert "overlaps" in text and "status 3" in text


def test_rows_apart_count_as_one_range(p):
    assert "overlaps" in message(p, logits_ld=2 * V, out_tokens=A + 4 * V)
    assert "overlaps" in message(p, logits_ld=2 * V, out_tokens=A + 4 * ((R * B - 1) * 2 * V + V) - 4)
    assert "overlaps" not in message(p, logits_ld=2 * V, out_tokens=A + 4 * ((R * B - 1) * 2 * V + V))
