"""The 64-bit restatement of the operators over a paged cache (plain_paged.py), against hand-worked examples and against forms that share nothing with it."""
import numpy as np

import plain_paged as P


def test_rotation_is_a_turn_of_channel_pairs():
    x = np.array([[1.0, 0.0, 2.0, 0.0, 7.0, 8.0]])
    row = np.zeros(6, dtype=np.float32)
    row[0:4] = [0.0, 1.0, -1.0, 0.0]   # pair 0 by a quarter, pair 1 by a half
    assert np.array_equal(P.rotated(x, row, 4, 0)[0], [[0.0, 1.0, -2.0, 0.0, 7.0, 8.0]])
    # pairs (0, 2) and (1, 3)
    assert np.array_equal(P.rotated(x, row, 4, 2)[0], [[-2.0, 0.0, 1.0, 0.0, 7.0, 8.0]])


def test_append_goes_through_the_table_and_leaves_the_rest():
    pages = np.zeros((3, 16, 1, 16))
    q = k = v = np.ones((4, 1, 16))
    tables = [[2, 0], [1]]
    qo, kp, vp, _, _, bad = P.append(pages, pages, tables, q, 2 * k, 3 * v, [17, -1, 16, 0], [0, 0, 1, 7], np.zeros((0, 16)), 0, 0)
    assert bad == 2                                   # sequence 1 has one page, sequence 7 none
    assert (kp[0, 1] == 2).all() and (vp[0, 1] == 3).all() and kp.sum() == 2 * 16
    assert (qo[0] == 1).all() and np.isnan(qo[1:]).all()


def test_attention_equals_a_softmax_over_gathered_positions():
    rng = np.random.default_rng(3)
    k, v = rng.standard_normal((2, 7, 16, 2, 8))
    tables = [[0, 1, 2], [6, 3, 4], [5, 5, 5]]
    q = rng.standard_normal((3, 4, 8))
    out, size, _, _ = P.attention(k, v, tables, q, [40, 33, 0], [20, 20, 20], [0, 3], 0.5, sinks=[0.0, 1.0, -np.inf, 2.0])
    for s, n in ((0, 40), (1, 33)):
        kk = np.stack([k[tables[0 if p < 20 else s][p // 16], p % 16] for p in range(n)])
        vv = np.stack([v[tables[0 if p < 20 else s][p // 16], p % 16] for p in range(n)])
        for h, sink in enumerate([0.0, 1.0, -np.inf, 2.0]):
            e = np.exp(kk[:, h // 2] @ q[s, h] * 0.5)
            assert np.allclose(out[s, h], e @ vv[:, h // 2] / (e.sum() + np.exp(sink)), rtol=1e-13, atol=1e-13)
    assert not out[2].any() and (size >= np.abs(out) - 1e-12).all()


def test_select_orders_by_score_then_beam_then_token():
    logits = np.log(np.array([[[0.5, 0.25, 0.25], [0.125, 0.125, 0.75]]]))
    s, w, b = P.select(logits, np.zeros((1, 2), dtype=np.float32), 4)
    assert list(w[0]) == [2, 0, 1, 2] and list(b[0]) == [1, 0, 0, 0]
    assert np.allclose(np.exp(s[0]), [0.75, 0.5, 0.25, 0.25])


def test_select_leaves_out_what_has_no_probability():
    nan, inf = np.nan, np.inf
    logits = np.array([[[nan, -inf, 3.0], [-inf, -inf, -inf], [1.0, 2.0, 3.0], [inf, 0.0, inf]]])
    s, w, b = P.select(logits, np.array([[-1.0, 0.0, -inf, -2.0]]), 6)
    assert list(w[0]) == [2, 0, 2, -1, -1, -1] and list(b[0]) == [0, 3, 3, -1, -1, -1]
    assert np.allclose(s[0, :3], [-1.0, -2.0 - np.log(2), -2.0 - np.log(2)]) and (s[0, 3:] == -inf).all()
    s, w, b = P.select(logits, np.array([[-1.0, 0.0, -3.0, -2.0]]), 2, done=np.array([[0, 0, 1, 1]]), end_token=1)
    assert list(w[0]) == [2, 1] and list(b[0]) == [0, 3] and list(s[0]) == [-1.0, -2.0]


def test_reorder_moves_only_second_children():
    pool = np.arange(8.0)[:, None]
    tables = [[0, 1, 4], [0, 2, 5], [0, 3, 6], [0, 7, 7]]
    t, n, row, pools = P.reorder([[2, 2, -1, 0]], tables, [20, 21, 22, 23], 16, [pool])
    assert row == [2, 1, 3, 0]                        # beam 1 takes row 1 (nobody continues 1 and 3), the idle beam row 3
    assert t == [tables[2], tables[1], tables[3], tables[0]] and n == [22, 22, 0, 20]
    assert list(pools[0][:, 0]) == [0, 1, 3, 3, 4, 5, 6, 7]   # page 2 became page 3; page 0 is shared, page 5 is behind 22 positions


def test_roundings_of_the_oracle():
    x = np.array([1.0 + 2.0 ** -9, 1.0 + 2.0 ** -8 + 2.0 ** -9, -3.14159])
    assert list(P.rounded(x, "BF16")[:2]) == [1.0, 1.0 + 2.0 ** -7]   # to even: 1 + 2^-8 + 2^-9 lies above the middle
    for ty in ("F16", "BF16"):
        y = P.rounded(x, ty)
        assert np.array_equal(P.values(P.bits(y, ty), ty), y) and (np.abs(y - x) <= P.HALF_STEP[ty] * np.abs(x)).all()
